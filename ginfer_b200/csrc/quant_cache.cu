// A key-value cache of 8 bits: rotation and quantised write of a step's keys and values, and reading
// them back.
//
// A row (the keys or the values of one token and kv head, `hd` channels) is kept as 8-bit codes and one
// 32-bit scale:
//     scale = max(amax |x| * (1/Q), 2^-126),  code = round_to_even(x * (1/scale)),  value = code * scale
// with Q = 127 (integers) or 448 (e4m3, saturating).  A row that holds an infinity or a NaN has no such
// codes: its scale is NaN and its codes are zero, so all of it reads back as NaN.  amax is taken before
// any rounding, so the codes stay in range whatever the row.
//
// Every product and sum of the rotation and the quantisation is rounded on its own (no fused
// multiply-add): a code follows from the formula alone, not from which kernel wrote it.
//
// Lay-out: codes [pages, kv heads, 2, page, hd] (keys, then values) and scales [pages, kv heads, page, 2].
// What one kv head keeps of a page is contiguous, and a token's two scales are one 8-byte word: the
// attention kernel reads a page's keys and values as one run.
#include "quant.cuh"

namespace gf {

// -------------------------------------------------------------------------------------- write
// A head's row is held by hd / 16 lanes of two times eight channels each, such that a lane's channels turn with
// each other: 8 l .. and half + 8 l .. where halves turn (what does not turn follows in runs of 16), 16 l .. where
// neighbours do.  A group of lanes takes HU heads of one token: their loads are under way together, and the angles
// of the token's position are read once for them.  What bounds it is reading the rows and writing q and the codes, each
// once; two heads a group with eight blocks an SM keep enough loads under way (launch_write: one head where the groups
// would not fill the SMs).
// Measured: 8,192 tokens of 28 + 2 x 4 heads of 128 in bfloat16, 143 MB: 29.5 us, 4.9 TB/s; one token: 3 us, a launch.
constexpr int WRITE_THREADS = 128;
// REGULAR: neighbours, or halves that are a multiple of eight.
template <typename T, int LANES, int HU, bool REGULAR>
__global__ void __launch_bounds__(WRITE_THREADS, REGULAR ? 8 : 6)
quant_write_kernel(const T* __restrict__ qkv, int row_stride, int tokens, int nh, int nkv, int hd,
                   const float* __restrict__ table, int table_rows, int rot, int neighbours,
                   const int* __restrict__ positions, const int* __restrict__ slots, T* __restrict__ q_out,
                   uint8_t* __restrict__ codes, int fp8, float* __restrict__ scales, int page, int num_slots,
                   int vec) {
  __shared__ float staged[REGULAR ? 1 : WRITE_THREADS * 17];
  pdl_trigger();
  pdl_wait();
  const int heads = nh + 2 * nkv;
  const int lane = threadIdx.x & (LANES - 1);
  // (a block's tokens all have the same heads: queries, keys or values, seldom two of them)
  const int t = blockIdx.x * (WRITE_THREADS / LANES) + threadIdx.x / LANES, h0 = blockIdx.y * HU;
  const bool here = t < tokens && lane * 16 < hd;
  const int half = rot >> 1;
  const bool plain = REGULAR && !neighbours;
  const bool turns = lane * 16 < rot;              // (all of a lane's channels, or with neighbours some)
  const int ca = plain && turns ? lane * 8 : lane * 16, cb = plain && turns ? half + lane * 8 : lane * 16 + 8;
  const T* row = qkv + (size_t)(here ? t : 0) * row_stride;
  const int slot = t < tokens ? fresh_index(slots + t) : -1;
  const bool keep = slot >= 0 && slot < num_slots;
  // the lanes of this row: groups of a warp part ways where one has queries and another keys
  const unsigned mask = (LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u)) << (threadIdx.x & 31 & ~(LANES - 1));

  Raw8<T> ra[HU], rb[HU];
#pragma unroll
  for (int i = 0; i < HU; ++i) {
    if (!here || h0 + i >= heads) continue;
    ra[i].load(row + (size_t)(h0 + i) * hd + ca, vec & 1);
    rb[i].load(row + (size_t)(h0 + i) * hd + cb, vec & 1);
  }
  const float* cs = table;
  float c[8], s[8];
  const int j0 = lane * 8;                         // the first of the lane's eight pairs
  if (here && rot > 0 && h0 < nh + nkv) {
    cs += (size_t)min(max(fresh_index(positions + t), 0), table_rows - 1) * rot;
    if (REGULAR && turns && (half & 7) == 0 && (vec & 2)) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {             // (a row of the table is a multiple of 64 bytes)
        const float4 cv = __ldg(reinterpret_cast<const float4*>(cs + j0 + e));
        const float4 sv = __ldg(reinterpret_cast<const float4*>(cs + half + j0 + e));
        c[e] = cv.x, c[e + 1] = cv.y, c[e + 2] = cv.z, c[e + 3] = cv.w;
        s[e] = sv.x, s[e + 1] = sv.y, s[e + 2] = sv.z, s[e + 3] = sv.w;
      }
    } else if (REGULAR && turns) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = min(j0 + e, half - 1);
        c[e] = __ldg(cs + j), s[e] = __ldg(cs + half + j);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HU; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;                         // (a group's lanes agree on h: the shuffles below are whole)
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.f;
    if (here) ra[i].get(lo), rb[i].get(hi);
    if (REGULAR && here && turns && h < nh + nkv) {
      if (plain) {
#pragma unroll
        for (int e = 0; e < 8; ++e) turn_pair(lo[e], hi[e], c[e], s[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (j0 + e < half) turn_pair(lo[2 * e], lo[2 * e + 1], c[e], s[e]);
          if (j0 + 4 + e < half) turn_pair(hi[2 * e], hi[2 * e + 1], c[4 + e], s[4 + e]);
        }
      }
    }
    if (!REGULAR && h < nh + nkv) {                // (halves that are no multiple of eight: partners through shared memory)
      float* mine = staged + threadIdx.x * 17;
      const float* first = staged + (threadIdx.x - lane) * 17;
#pragma unroll
      for (int e = 0; e < 8; ++e) mine[e] = lo[e], mine[8 + e] = hi[e];
      __syncwarp(mask);
      if (here) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int ch = lane * 16 + e;
          float& own = e < 8 ? lo[e & 7] : hi[e & 7];
          if (ch >= rot) continue;
          const int j = ch < half ? ch : ch - half, other = ch < half ? ch + half : j;
          const float o = first[(other >> 4) * 17 + (other & 15)];
          own = ch < half ? turned_first(own, o, __ldg(cs + j), __ldg(cs + half + j))
                          : turned_second(o, own, __ldg(cs + j), __ldg(cs + half + j));
        }
      }
      __syncwarp(mask);
    }
    if (h < nh) {
      if (here) {
        T* q = q_out + (size_t)t * nh * hd + (size_t)h * hd;
        store8(q + ca, lo);
        store8(q + cb, hi);
      }
      continue;
    }
    const uint32_t top = group_max_bits<LANES>(max(max_bits8(lo), max_bits8(hi)), mask);
    if (!keep) continue;
    const int which = h >= nh + nkv, kvh = h - nh - which * nkv;
    const RowScale rs = row_scale(top, fp8);
    const int pg = slot / page, off = slot - pg * page;
    const size_t at = (size_t)pg * nkv + kvh;
    uint8_t* dst = codes + ((at * 2 + which) * page + off) * hd;
    if (here) {
      *reinterpret_cast<uint2*>(dst + ca) = quantise8(lo, rs, fp8);
      *reinterpret_cast<uint2*>(dst + cb) = quantise8(hi, rs, fp8);
    }
    if (lane == 0) scales[(at * page + off) * 2 + which] = rs.scale;
  }
}

template <typename T, int LANES>
int launch_write(const void* qkv, int row_stride, int tokens, int nh, int nkv, int hd, const float* table,
                 int table_rows, int rot, int neighbours, const int* positions, const int* slots, void* q_out,
                 uint8_t* codes, int fp8, float* scales, int page, int num_slots, int vec, int sms,
                 cudaStream_t stream) {
  const int heads = nh + 2 * nkv;
  // One head a group while that is at most two rounds of 1,024 threads an SM: more groups, so that loads are under way
  // everywhere; beyond it, two heads read a position's angles once.  One / two, us: 28 + 2 x 4 heads of 128 in bfloat16 at a
  // quarter round 2.9 / 3.4, one round (526 tokens) 3.8 / 4.6, two 5.6 / 5.6, three 7.5 / 7.4, eight 18.7 / 16.3; 14 + 2 x 2 of 64
  // 4.0 / 4.9 at one, 5.9 / 6.0 at two, 8.1 / 8.2 at three, 20.6 / 17.8 at eight; 12 + 2 x 2 of 128 in 32 bits 8.2 / 8.5 at two,
  // 12.0 / 13.0 at three, 28.0 / 27.9 at eight.
  const bool one = (long long)tokens * heads * LANES <= 2048LL * sms;
  const int hu = one ? 1 : 2, sets = (heads + hu - 1) / hu, each = WRITE_THREADS / LANES;
  if (sets > 65535) return -5;
  const dim3 grid((unsigned)((tokens + each - 1) / each), (unsigned)sets);
  const auto run = [&](auto kernel) {
    return launch_kernel(kernel, grid, dim3(WRITE_THREADS), 0, stream, (const T*)qkv, row_stride,
                         tokens, nh, nkv, hd, table, table_rows, rot, neighbours, positions, slots, (T*)q_out,
                         codes, fp8, scales, page, num_slots, vec);
  };
  if (neighbours || rot % 16 == 0)
    return one ? run(quant_write_kernel<T, LANES, 1, true>) : run(quant_write_kernel<T, LANES, 2, true>);
  return one ? run(quant_write_kernel<T, LANES, 1, false>) : run(quant_write_kernel<T, LANES, 2, false>);
}

// -------------------------------------------------------------------------------------- read
// Dense [2, B, S, kv heads, hd]: position s of request b through its block table where first <= s < length,
// zeros elsewhere; or, with `slots`, row s of [2, 1, S, kv heads, hd] from slot slots[s] (negative: zeros).
// A block takes READ_SPAN positions and works out where they lie once; a thread keeps its 16 bytes' place in a
// token's result and walks down the positions, four loads under way.  What bounds it is writing the result, twice
// (32-bit: four times) the bytes that it reads.  Small blocks, many an SM, so that one block's look-ups pass under
// the others' copies; of twice the threads where a token's result is twice the bytes.
// Measured: two requests, 32,768 positions wide, 4 kv heads of 128 in bfloat16, 50 MB to 134 MB: 34.1 us, 5.4 TB/s (with
// blocks of 256 threads 36.6, of 32 positions 37.6); 7 of 3,040, windows of 1,024, 5 heads of 80 in 32 bits: 16.4 us (with
// blocks of 128 threads 20.5).
constexpr int READ_SPAN = 16;
template <typename T> constexpr int READ_THREADS = 64 * (int)sizeof(T);
template <typename T>
__global__ void __launch_bounds__(READ_THREADS<T>, 24 / (int)sizeof(T))
quant_read_kernel(const uint8_t* __restrict__ codes, int fp8, const float* __restrict__ scales,
                  const int* __restrict__ block_table, int table_stride, const int* __restrict__ lengths,
                  const int* __restrict__ first, const int* __restrict__ slots, int num_slots, int S, int nkv,
                  int hd, int page, T* __restrict__ out) {
  constexpr int E = 16 / (int)sizeof(T);             // channels of a thread
  __shared__ int2 token_at[READ_SPAN];               // page number (-1: zeros), place
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, s0 = blockIdx.x * READ_SPAN, num_pages = num_slots / page;
  if (threadIdx.x < READ_SPAN) {
    const int s = s0 + threadIdx.x;
    int pg = -1, off = 0;
    if (s < S) {
      if (slots) {
        const int slot = fresh_index(slots + s);
        if (slot >= 0 && slot < num_slots) pg = slot / page, off = slot - pg * page;
      } else if (s < fresh_index(lengths + b) && (!first || s >= fresh_index(first + b))) {
        const int lp = s / page;
        pg = min(max(fresh_index(block_table + (size_t)b * table_stride + lp), 0), num_pages - 1), off = s - lp * page;
      }
    }
    token_at[threadIdx.x] = make_int2(pg, off);
  }
  __syncthreads();
  const int chunks = hd / E, units = 2 * nkv * chunks;
  // threads side by side in a token's result, and as many tokens at a time as then fit the block
  const int wide = min(units, READ_THREADS<T>), deep = READ_THREADS<T> / wide;
  const int down = threadIdx.x / wide;
  if (down >= deep) return;
  const int many = min(READ_SPAN, S - s0);
  for (int u = threadIdx.x - down * wide; u < units; u += wide) {
    const int which = u >= nkv * chunks, v = u - which * nkv * chunks, kvh = v / chunks, ch = v - kvh * chunks;
    T* to = out + ((((size_t)which * gridDim.y + b) * S + s0) * nkv + kvh) * hd + ch * E;
    const size_t step = (size_t)nkv * hd;
    for (int d0 = down; d0 < many; d0 += 4 * deep) {
      uint32_t raw[4][E / 4];
      float sc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d0 + i * deep;
        const int2 at = d < many ? token_at[d] : make_int2(-1, 0);
        sc[i] = 0.f;
#pragma unroll
        for (int e = 0; e < E / 4; ++e) raw[i][e] = 0u;
        if (at.x >= 0) {
          const size_t record = (size_t)at.x * nkv + kvh;
          const uint8_t* from = codes + ((record * 2 + which) * page + at.y) * hd + ch * E;
          if constexpr (E == 8) {
            const uint2 r = __ldcg(reinterpret_cast<const uint2*>(from));
            raw[i][0] = r.x, raw[i][1] = r.y;
          } else {
            raw[i][0] = __ldcg(reinterpret_cast<const uint32_t*>(from));
          }
          sc[i] = __ldcg(scales + (record * page + at.y) * 2 + which);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d0 + i * deep;
        if (d >= many) continue;
        float x[E];
#pragma unroll
        for (int e = 0; e < E / 4; ++e) values4(raw[i][e], fp8, x + 4 * e);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = token_at[d].x < 0 ? 0.f : __fmul_rn(x[e], sc[i]);
        T* o = to + (size_t)d * step;
        if constexpr (E == 8) store8(o, x);
        else *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
  }
}

}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// qkv [T, >= (nh + 2 nkv) hd] with `row_stride`; table [table_rows, rot] fp32 (cosines, sines) or null with
// rot 0; q_out [T, nh hd].  A slot outside the cache is not written, a position outside the table takes its
// nearest row.
struct WriteCall {
  const void* qkv;
  long long row_stride, dtype, tokens, nh, nkv, hd;
  const float* table;
  long long table_rows, rot, neighbours;
  const int *positions, *slots;
  void *q_out, *codes;
  long long fp8;
  float* scales;
  long long page, pages;
  cudaStream_t stream;
  long long sms;
};
static_assert(sizeof(WriteCall) == 21 * 8, "the caller packs it");

GF_EXPORT int gf_quant_write(const WriteCall* call) {
  const WriteCall& c = *call;
  if (c.tokens <= 0) return c.tokens < 0 ? -3 : 0;
  if (c.hd % 16 || c.hd < 16 || c.hd > 256 || c.nh < 1 || c.nkv < 1 || c.nh > 1 << 20 || c.nkv > 1 << 20 || c.page < 1 ||
      c.pages < 0 || c.page * c.pages > 0x7fffffffLL || c.rot < 0 || c.rot % 2 || c.rot > c.hd ||
      (c.rot && (!c.table || c.table_rows < 1)) || c.tokens > 0x7fffffff || c.row_stride > 0x7fffffff || c.row_stride < 0 || c.sms < 1 || c.sms > 1 << 20)
    return -3;
  const size_t es = c.dtype == GF_F32 ? 4 : 2;
  if ((size_t)c.codes % 16 || (size_t)c.scales % 8) return -3;
  // whether rows (1) and the table (2) can be read 16 bytes at a time
  const int vec = ((size_t)c.qkv % 16 == 0 && (size_t)c.row_stride * es % 16 == 0 ? 1 : 0) |
                  ((size_t)c.table % 16 == 0 ? 2 : 0);
  const auto go = [&](auto tag) {
    using T = decltype(tag);
    const auto run = [&](auto launch) {
      return launch(c.qkv, (int)c.row_stride, (int)c.tokens, (int)c.nh, (int)c.nkv, (int)c.hd, c.table, (int)c.table_rows,
                    (int)c.rot, c.neighbours != 0, c.positions, c.slots, c.q_out, (uint8_t*)c.codes, (int)c.fp8, c.scales,
                    (int)c.page, (int)(c.page * c.pages), vec, (int)c.sms, c.stream);
    };
    if (c.hd <= 64) return run(launch_write<T, 4>);
    if (c.hd <= 128) return run(launch_write<T, 8>);
    return run(launch_write<T, 16>);
  };
  return c.dtype == GF_F32 ? go(float()) : go(bf16());
}

// block_table, lengths (and first, may be null) of B requests, out [2, B, S, nkv, hd]; or slots [S] with B = 1.
struct ReadCall {
  const void* codes;
  long long fp8;
  const float* scales;
  const int* block_table;
  long long table_stride;
  const int *lengths, *first, *slots;
  long long pages, B, S, nkv, hd, page;
  void* out;
  long long dtype;
  cudaStream_t stream;
};
static_assert(sizeof(ReadCall) == 17 * 8, "the caller packs it");

GF_EXPORT int gf_quant_read(const ReadCall* call) {
  const ReadCall& c = *call;
  if (c.B <= 0 || c.S <= 0) return c.B < 0 || c.S < 0 ? -3 : 0;
  if (c.hd % 16 || c.hd < 16 || c.hd > 256 || c.nkv < 1 || c.nkv > 1 << 20 || c.page < 1 || c.pages < 0 ||
      c.page * c.pages > 0x7fffffffLL || c.B > 65535 || c.S > 0x7fffffff - READ_SPAN || c.table_stride > 0x7fffffff ||
      (size_t)c.codes % 16)
    return -3;
  const dim3 grid((unsigned)((c.S + READ_SPAN - 1) / READ_SPAN), (unsigned)c.B);
  const auto go = [&](auto tag) {
    using T = decltype(tag);
    return launch_kernel(quant_read_kernel<T>, grid, dim3(READ_THREADS<T>), 0, c.stream,
                         (const uint8_t*)c.codes, (int)c.fp8, c.scales, c.block_table, (int)c.table_stride, c.lengths,
                         c.first, c.slots, (int)(c.page * c.pages), (int)c.S, (int)c.nkv, (int)c.hd, (int)c.page,
                         (T*)c.out);
  };
  return c.dtype == GF_F32 ? go(float()) : go(bf16());
}
