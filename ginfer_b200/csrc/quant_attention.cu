// One new token's attention over a paged key-value cache of 8 bits (quant_cache.cu: its formulas and
// lay-out), compiled for one head size (-DGF_HEAD_DIM=<multiple of 16, at most 256>).
//
// For a request of `len` tokens the query is the last one, at position p = len - 1; it sees the keys
// first_visible_key(p, span) .. p.  out = sum_c softmax_c(scale <q, K_c>) V_c; a request without a
// token gives zeros.
//
// What bounds it is reading the cache: 2 HD + 8 bytes a key and kv head, used once.  So a code goes from
// memory to the registers of the one thread that multiplies it, without shared memory between:
//
//  * S^T = K q^T on mma.sync.m16n8k16 (half precision in, 32-bit sums): 16 keys are the rows, up to 8 query
//    heads of a kv head the columns.  The order of a product's reduction is free as long as both operands
//    share it, so the channels are dealt to the instruction's places such that a thread's places are
//    neighbours in memory: it loads up to 16 bytes of its two keys at a time.
//  * O^T = V^T P^T: the rows are channels, the reduction runs over the 16 keys.  A thread's rows are again
//    chosen to be neighbours in memory; two keys' codes of a channel are put side by side by a byte
//    permutation.  P^T comes from S^T by movmatrix.
//  * Codes become halves exactly: e4m3 by one conversion of two, int8 as 1024 + 128 + code, whose bits are
//    0x64 above the code's, minus 1152.
//
// Half precision holds q and the weights in 11 bits (a row of q is scaled by a power of two so that its
// largest element is in [2^14, 2^15); a weight, p times its value row's scale, so that the largest value
// scale seen so far gives [2^14, 2^15)): more than the 8 bits of a bfloat16 q and result.  For 32-bit q both
// are the sum of two halves (22 bits), and tiles' products are added up outside the tensor cores.  Scores,
// maxima, sums and O are 32-bit.
//
// The work is cut into pieces of equal numbers of 16-key tiles, whatever the requests' lengths: see
// find_piece.  A piece is a block of four warps, which take its tiles in turn.  Where a request has several
// pieces, they leave their results (normalised, with maximum and sum) in scratch, and a second kernel joins
// them in order.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "quant.cuh"

#ifndef GF_HEAD_DIM
#define GF_HEAD_DIM 128
#endif

namespace gf {

constexpr int HD = GF_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16, <= 256");
constexpr float kLog2E = 1.4426950408889634f;
constexpr int TILE = 16, WARPS = 4, THREADS = WARPS * 32;
constexpr int KW = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4;     // bytes of a key a thread loads at once
constexpr int VW = HD % 128 == 0 ? 16 : HD % 64 == 0 ? 8 : HD % 32 == 0 ? 4 : 2;
constexpr int KWORDS = HD / 16;                                  // words of a key a thread holds
constexpr int VWORDS = VW >= 4 ? HD / 32 : HD / 16;              // of a value (2-byte loads: a word each)
constexpr int MT = HD / 16;                                      // row tiles of O^T
// values of the next tile are loaded a tile ahead like its keys, where registers allow
constexpr bool kValuesAhead = HD <= 128;
// the fewest tiles a piece is worth
constexpr int kLeastTiles = 8 * WARPS;
constexpr int kMostBlocks = 8;          // of the blocks that fit an SM, so many are counted on

struct DecodeArgs {
  const void* q;              // rows of q, or of q | k | v (fused)
  int q_stride, q_f32;
  uint8_t* codes;
  float* scales;
  const int* block_table;
  int table_stride, limit;    // limit: no request is longer (table width * page)
  const int* lengths;
  void* out;
  int out_f32, B, nh, nkv, page, page_shift, span;
  float scale;
  int chunks, rows;           // a kv head's query heads in `chunks` blocks of up to `rows`
  int slots;                  // blocks that fit the GPU at once
  float* po;                  // [pieces * heads][rows][HD]
  float2* pml;                // [pieces * heads][rows]
  // the fused step
  const float* table;
  int table_rows, rot, neighbours;
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------------------------- division of the work
// Request b has n_b tiles (positions first_visible .. len - 1, cut at multiples of 16).  With room for N
// pieces a kv head at once (N = slots / heads) a piece holds at most
//     size = sum n_b / (N - B + 1) tiles   where 2 B <= N: then all pieces run at once
//     size = sum n_b heads / (2 slots)     else: two rounds and the requests' remainders even out
// and request b has max(1, n_b / size rounded up) pieces.  Every warp of a block works this out for itself.
struct Piece {
  int b, first, last, lo, len;    // tiles [first, last) of request b; its keys are lo .. len - 1
  int pieces, index;              // how many pieces b has, which this is
};
__device__ __forceinline__ int request_length(const DecodeArgs& a, int b) {
  return max(min(fresh_index(a.lengths + b), a.limit), 0);
}
__device__ __forceinline__ int request_tiles(const DecodeArgs& a, int len) {
  return len > 0 ? ((len - 1) >> 4) - (first_visible_key(len - 1, a.span) >> 4) + 1 : 0;
}
__device__ __forceinline__ int piece_size(const DecodeArgs& a, int lane) {
  long long total = 0;
  for (int b = lane; b < a.B; b += 32) total += request_tiles(a, request_length(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const int heads = a.nkv * a.chunks, N = a.slots / heads;
  const long long size = 2 * a.B <= N ? (total + N - a.B) / (N - a.B + 1)
                                      : (total * heads + 2 * a.slots - 1) / (2 * a.slots);
  return (int)max(size, (long long)kLeastTiles);
}
// The piece with number `want` in the order of the requests; b = -1: there are fewer.
__device__ __forceinline__ Piece find_piece(const DecodeArgs& a, int want, int lane) {
  const int size = piece_size(a, lane);
  Piece r;
  r.b = -1;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    const int len = b < a.B ? request_length(a, b) : 0;
    const int n = request_tiles(a, len);
    const int mine = b < a.B ? max(1, (n + size - 1) / size) : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int start = before + sum - mine;
    const unsigned hit = __ballot_sync(0xffffffffu, want >= start && want < start + mine);
    if (hit) {
      const int src = __ffs(hit) - 1;
      r.b = b0 + src;
      r.len = __shfl_sync(0xffffffffu, len, src);
      r.pieces = __shfl_sync(0xffffffffu, mine, src);
      r.index = want - __shfl_sync(0xffffffffu, start, src);
      const int tiles = __shfl_sync(0xffffffffu, n, src);
      r.lo = r.len > 0 ? first_visible_key(r.len - 1, a.span) : 0;
      const int t0 = r.lo >> 4;
      r.first = t0 + min(r.index * size, tiles);
      r.last = t0 + min((r.index + 1) * size, tiles);
      return r;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return r;
}

// ------------------------------------------------------------------------------------- a tile
struct Tile {
  uint32_t k[2][KWORDS];      // keys g and g + 8: channels as the thread's places want them
  uint32_t v[4][VWORDS];      // keys 2t, 2t + 1, 2t + 8, 2t + 9
  float2 sc[2];               // (key, value) scales of keys g and g + 8
};
template <int BYTES> __device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* r);
template <> __device__ __forceinline__ void load_bytes<16>(const uint8_t* p, uint32_t* r) {
  const uint4 x = __ldcg(reinterpret_cast<const uint4*>(p));
  r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
}
template <> __device__ __forceinline__ void load_bytes<8>(const uint8_t* p, uint32_t* r) {
  const uint2 x = __ldcg(reinterpret_cast<const uint2*>(p));
  r[0] = x.x, r[1] = x.y;
}
template <> __device__ __forceinline__ void load_bytes<4>(const uint8_t* p, uint32_t* r) {
  r[0] = __ldcg(reinterpret_cast<const uint32_t*>(p));
}
template <> __device__ __forceinline__ void load_bytes<2>(const uint8_t* p, uint32_t* r) {
  r[0] = __ldcg(reinterpret_cast<const unsigned short*>(p));
}
__device__ __forceinline__ void load_key(const uint8_t* row, int t, uint32_t (&r)[KWORDS]) {
#pragma unroll
  for (int j = 0; j < HD / (4 * KW); ++j) load_bytes<KW>(row + (j * 4 + t) * KW, r + j * (KW / 4));
}
__device__ __forceinline__ void load_value(const uint8_t* row, int g, uint32_t (&r)[VWORDS]) {
  constexpr int STEP = VW >= 4 ? VW / 4 : 1;
#pragma unroll
  for (int j = 0; j < HD / (8 * VW); ++j) load_bytes<VW>(row + (j * 8 + g) * VW, r + j * STEP);
}
// Where a key lies.  WHOLE: pages are a multiple of the tile, a tile has one page.
struct Place {
  const uint8_t* codes;       // the key's row; its value's lies page * HD behind
  const float2* scales;
};
__device__ __forceinline__ Place place_of(const DecodeArgs& a, int kvh, int page_number, int off) {
  const size_t at = (size_t)page_number * a.nkv + kvh;
  return {a.codes + (at * 2 * a.page + off) * HD, reinterpret_cast<const float2*>(a.scales) + at * a.page + off};
}
__device__ __forceinline__ int logical_page(const DecodeArgs& a, int c) {
  return a.page_shift >= 0 ? c >> a.page_shift : c / a.page;
}
__device__ __forceinline__ Place place_of_key(const DecodeArgs& a, const Piece& pc, int kvh, int c) {
  c = min(max(c, pc.lo), pc.len - 1);            // (a masked key: any that is there)
  const int lp = logical_page(a, c);
  return place_of(a, kvh, fresh_index(a.block_table + (size_t)pc.b * a.table_stride + lp), c - lp * a.page);
}
template <bool WHOLE, bool KEYS, bool VALUES>
__device__ __forceinline__ void load_tile(Tile& x, const DecodeArgs& a, const Piece& pc, int kvh, int tile,
                                          int page_number, int g, int t) {
  const int c0 = tile * TILE;
  if constexpr (WHOLE) {
    const Place p = place_of(a, kvh, page_number, c0 - logical_page(a, c0) * a.page);
    if constexpr (KEYS) {
      load_key(p.codes + g * HD, t, x.k[0]);
      load_key(p.codes + (g + 8) * HD, t, x.k[1]);
      x.sc[0] = __ldcg(p.scales + g);
      x.sc[1] = __ldcg(p.scales + g + 8);
    }
    if constexpr (VALUES) {
      const uint8_t* v = p.codes + (size_t)a.page * HD + 2 * t * HD;
      load_value(v, g, x.v[0]);
      load_value(v + HD, g, x.v[1]);
      load_value(v + 8 * HD, g, x.v[2]);
      load_value(v + 9 * HD, g, x.v[3]);
    }
  } else {
    if constexpr (KEYS) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Place p = place_of_key(a, pc, kvh, c0 + g + 8 * i);
        load_key(p.codes, t, x.k[i]);
        x.sc[i] = __ldcg(p.scales);
      }
    }
    if constexpr (VALUES) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_value(place_of_key(a, pc, kvh, c0 + 2 * t + (i & 1) + 8 * (i >> 1)).codes + (size_t)a.page * HD, g,
                   x.v[i]);
    }
  }
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
// 2^(127 - f) for 14 <= f <= 254
__device__ __forceinline__ float power_back(int f) {
  return __uint_as_float(f == 254 ? 0x00400000u : (uint32_t)(254 - f) << 23);
}

// ------------------------------------------------------------------------------------- q, and the new token
// Channel c of head row x at the token's position.
__device__ __forceinline__ float row_value(const DecodeArgs& a, size_t at, int c) {
  return a.q_f32 ? fresh(reinterpret_cast<const float*>(a.q) + at + c)
                 : fresh(reinterpret_cast<const bf16*>(a.q) + at + c);
}
__device__ __forceinline__ float rotated_value(const DecodeArgs& a, size_t at, int c, const float* cs) {
  const float x = row_value(a, at, c);
  if (c >= a.rot) return x;
  const int half = a.rot >> 1;
  const bool second = a.neighbours ? (c & 1) : c >= half;
  const int j = a.neighbours ? c >> 1 : second ? c - half : c;
  const float o = row_value(a, at, a.neighbours ? c ^ 1 : second ? c - half : c + half);
  return second ? turned_second(o, x, cs[j], cs[half + j]) : turned_first(x, o, cs[j], cs[half + j]);
}

// ------------------------------------------------------------------------------------- a piece
// NT: tiles of 8 query heads.  PARTS: halves that make up q and a weight.  STEP: q | k | v rows, unrotated.
template <int NT, bool FP8, int PARTS, bool WHOLE, bool STEP>
__global__ void __launch_bounds__(THREADS, (NT == 1 && HD <= 128 && PARTS == 1) ? 3 : 2)
quant_decode_kernel(const DecodeArgs a) {
  constexpr int R = 8 * NT, N = (HD + 31) / 32;
  extern __shared__ __align__(16) float so[];                    // [WARPS][R][HD], at the end
  __shared__ __align__(16) __half qh[PARTS][R][HD];
  __shared__ float qs[R], sm[WARPS][R], sl[WARPS][R], ww[WARPS][R], total[R];
  pdl_trigger();
  pdl_wait();
  const int heads = a.nkv * a.chunks;
  const int hc = blockIdx.x % heads, kvh = hc / a.chunks, chunk = hc - kvh * a.chunks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Piece pc = find_piece(a, blockIdx.x / heads, lane);
  if (pc.b < 0) return;
  const int G = a.nh / a.nkv, h0 = kvh * G + chunk * a.rows, nrows = min(a.rows, G - chunk * a.rows);
  if (pc.len <= 0) {
    for (int i = threadIdx.x; i < nrows * HD; i += THREADS) {
      const size_t at = ((size_t)pc.b * a.nh + h0) * HD + i;
      if (a.out_f32) reinterpret_cast<float*>(a.out)[at] = 0.f;
      else reinterpret_cast<bf16*>(a.out)[at] = __float2bfloat16_rn(0.f);
    }
    return;
  }
  const int* tbl = a.block_table + (size_t)pc.b * a.table_stride;
  const size_t row = (size_t)pc.b * a.q_stride;
  const int p = pc.len - 1;
  const float* cs = nullptr;
  if constexpr (STEP) cs = a.table + (size_t)min(p, a.table_rows - 1) * a.rot;

  if constexpr (STEP) {
    // The new token's row of keys and of values: the piece that holds it writes it (every chunk of heads the
    // same bytes) and reads it back with its tile.
    if (pc.index == pc.pieces - 1 && warp < 2) {
      const size_t at = row + (size_t)(a.nh + warp * a.nkv + kvh) * HD;
      float x[N];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = i * 32 + lane;
        x[i] = c >= HD ? 0.f : warp == 0 ? rotated_value(a, at, c, cs) : row_value(a, at, c);
        top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
      }
      const RowScale rs = row_scale(group_max_bits<32>(top), FP8);
      const int lp = logical_page(a, p), off = p - lp * a.page;
      const Place pl = place_of(a, kvh, fresh_index(tbl + lp), off);
      uint8_t* dst = const_cast<uint8_t*>(pl.codes) + (size_t)warp * a.page * HD;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i * 32 + lane < HD) dst[i * 32 + lane] = (uint8_t)code_of(x[i], rs, FP8);
      if (lane == 0) reinterpret_cast<float*>(const_cast<float2*>(pl.scales))[warp] = rs.scale;
    }
  }
  // q in halves, a row's largest element in [2^14, 2^15)
  for (int r = warp; r < R; r += WARPS) {
    const size_t at = row + (size_t)(h0 + r) * HD;
    float x[N];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * 32 + lane;
      x[i] = r >= nrows || c >= HD ? 0.f : STEP ? rotated_value(a, at, c, cs) : row_value(a, at, c);
      top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    top = group_max_bits<32>(top);
    // 2^up takes the largest element to [2^14, 2^15); what is no number stays none
    const int e = top >= 0x7f800000u ? 127 : max((int)(top >> 23), 1), up = min(127 + 14 - e, 126);
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * 32 + lane;
      if (c < HD) {
        qh[0][r][c] = __float2half_rn(x[i] * f);
        if constexpr (PARTS == 2) qh[1][r][c] = __float2half_rn(half_rest(x[i] * f));
      }
    }
    if (lane == 0) qs[r] = a.scale * kLog2E * __uint_as_float((uint32_t)(127 - up) << 23);
  }
  __syncthreads();

  uint32_t qf[PARTS][NT][KWORDS][2];
#pragma unroll
  for (int w = 0; w < KWORDS; ++w) {
    constexpr int STEPS = KW / 4;
    const int c = ((w / STEPS) * 4 + t) * KW + (w % STEPS) * 4;      // the channels of a key's word w
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const uint2 two = *reinterpret_cast<const uint2*>(&qh[i][n * 8 + g][c]);
        qf[i][n][w][0] = two.x, qf[i][n][w][1] = two.y;
      }
  }
  float qscale[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) qscale[n][0] = qs[n * 8 + 2 * t], qscale[n][1] = qs[n * 8 + 2 * t + 1];

  float o[NT][MT][4], m[NT][2], l[NT][2];
  int f = 254;               // weights are multiplied by 2^(f - 127)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }
  const auto page_at = [&](int tile) {
    return WHOLE && tile < pc.last ? fresh_index(tbl + logical_page(a, tile * TILE)) : 0;
  };
  const auto work = [&](Tile& x, int tile) {
    const int c0 = tile * TILE;
    const bool edge = c0 < pc.lo || c0 + TILE > pc.len;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int w = 0; w < KWORDS; ++w) {
      const uint32_t k0 = FP8 ? x.k[0][w] : x.k[0][w] ^ 0x80808080u, k1 = FP8 ? x.k[1][w] : x.k[1][w] ^ 0x80808080u;
      const uint32_t A[4] = {halves<FP8>(k0, 0), halves<FP8>(k1, 0), halves<FP8>(k0, 1), halves<FP8>(k1, 1)};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) mma_f16(s[n], A, qf[i][n][w][0], qf[i][n][w][1]);
    }
    float2 sc[2] = {x.sc[0], x.sc[1]};
    bool seen[2] = {true, true};
    if (edge) {
      // masked keys: whatever lies there counts as nothing
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = c0 + g + 8 * i;
        seen[i] = c >= pc.lo && c < pc.len;
        if (!seen[i]) sc[i] = make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 2 * t + (i & 1) + 8 * (i >> 1);
        if (c < pc.lo || c >= pc.len)
#pragma unroll
          for (int w = 0; w < VWORDS; ++w) x.v[i][w] = 0u;
      }
    }
    float mn[NT][2];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[n][j] = seen[0] ? s[n][j] * sc[0].x * qscale[n][j] : -INFINITY;
        s[n][2 + j] = seen[1] ? s[n][2 + j] * sc[1].x * qscale[n][j] : -INFINITY;
        float top = fmaxf(s[n][j], s[n][2 + j]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        mn[n][j] = fmaxf(m[n][j], top);
        moved |= mn[n][j] != m[n][j];
      }
    const uint32_t b0 = __float_as_uint(sc[0].y), b1 = __float_as_uint(sc[1].y);
    const uint32_t vtop = __reduce_max_sync(0xffffffffu, max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u));
    const int fn = min(f, 127 + 14 + 127 - (int)(vtop >> 23));
    if (__any_sync(0xffffffffu, moved) || fn != f) {
      const float back = fn == f ? 1.f : f - fn > 126 ? 0.f : __uint_as_float((uint32_t)(127 + fn - f) << 23);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float corr[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          corr[j] = mn[n][j] == m[n][j] ? 1.f : fast_exp2(m[n][j] - mn[n][j]);
          l[n][j] *= corr[j];
          corr[j] *= back;
          m[n][j] = mn[n][j];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
          o[n][i][0] *= corr[0], o[n][i][1] *= corr[1], o[n][i][2] *= corr[0], o[n][i][3] *= corr[1];
      }
      f = fn;
    }
    const float up = __uint_as_float((uint32_t)f << 23);
    const float vs0 = sc[0].y * up, vs1 = sc[1].y * up;
    uint32_t P[PARTS][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float w[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p0 = fast_exp2(s[n][j] - m[n][j]), p1 = fast_exp2(s[n][2 + j] - m[n][j]);
        l[n][j] += p0 + p1;
        w[j] = p0 * vs0, w[2 + j] = p1 * vs1;
      }
      P[0][n][0] = transposed(pack_half(w[0], w[1]));
      P[0][n][1] = transposed(pack_half(w[2], w[3]));
      if constexpr (PARTS == 2) {
        P[1][n][0] = transposed(pack_half(half_rest(w[0]), half_rest(w[1])));
        P[1][n][1] = transposed(pack_half(half_rest(w[2]), half_rest(w[3])));
      }
    }
    const auto add = [&](int i, const uint32_t (&A)[4]) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (PARTS == 2) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(d, A, P[1][n][0], P[1][n][1]);
          mma_f16(d, A, P[0][n][0], P[0][n][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][i][e] += d[e];
        } else {
          mma_f16(o[n][i], A, P[0][n][0], P[0][n][1]);
        }
      }
    };
#pragma unroll
    for (int w = 0; w < VWORDS; ++w) {
      if constexpr (!FP8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i][w] ^= 0x80808080u;
      }
      const uint32_t u0 = __byte_perm(x.v[0][w], x.v[1][w], 0x5140), u1 = __byte_perm(x.v[2][w], x.v[3][w], 0x5140);
      const uint32_t A[4] = {halves<FP8>(u0, 0), halves<FP8>(u0, 1), halves<FP8>(u1, 0), halves<FP8>(u1, 1)};
      if constexpr (VW >= 4) {
        add(2 * w, A);
        const uint32_t y0 = __byte_perm(x.v[0][w], x.v[1][w], 0x7362);
        const uint32_t y1 = __byte_perm(x.v[2][w], x.v[3][w], 0x7362);
        const uint32_t C[4] = {halves<FP8>(y0, 0), halves<FP8>(y0, 1), halves<FP8>(y1, 0), halves<FP8>(y1, 1)};
        add(2 * w + 1, C);
      } else {
        add(w, A);
      }
    }
  };

  int tile = pc.first + warp;
  if (tile < pc.last) {
    Tile x, y;
    const int pg0 = page_at(tile);
    int pg = page_at(tile + WARPS);
    load_tile<WHOLE, true, kValuesAhead>(x, a, pc, kvh, tile, pg0, g, t);
    int pg_x = pg0;
    while (true) {
      const int next = tile + WARPS;
      const int pg_y = pg;
      if constexpr (!kValuesAhead) load_tile<WHOLE, false, true>(x, a, pc, kvh, tile, pg_x, g, t);
      if (next < pc.last) {
        load_tile<WHOLE, true, kValuesAhead>(y, a, pc, kvh, next, pg_y, g, t);
        pg = page_at(next + WARPS);
      }
      work(x, tile);
      if (next >= pc.last) break;
      tile = next + WARPS;
      pg_x = pg;
      if constexpr (!kValuesAhead) load_tile<WHOLE, false, true>(y, a, pc, kvh, next, pg_y, g, t);
      if (tile < pc.last) {
        load_tile<WHOLE, true, kValuesAhead>(x, a, pc, kvh, tile, pg_x, g, t);
        pg = page_at(tile + WARPS);
      }
      work(y, next);
      if (tile >= pc.last) break;
    }
  }

  // the four warps' results
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
      l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
      l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
      if (g == 0) sm[warp][n * 8 + 2 * t + j] = m[n][j], sl[warp][n * 8 + 2 * t + j] = l[n][j];
    }
    constexpr int STEP_W = VW >= 4 ? VW / 4 : 1, PER = VW >= 4 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int w = i / PER;
      const int c = ((w / STEP_W) * 8 + g) * VW + (w % STEP_W) * 4 + (i % PER) * 2;
      float* at = so + ((size_t)warp * R + n * 8 + 2 * t) * HD + c;
      *reinterpret_cast<float2*>(at) = make_float2(o[n][i][0], o[n][i][2]);
      *reinterpret_cast<float2*>(at + HD) = make_float2(o[n][i][1], o[n][i][3]);
    }
  }
  if (lane == 0) ww[warp][0] = power_back(f);
  __syncthreads();
  float back = 0.f;
  if (threadIdx.x < WARPS * R) back = ww[threadIdx.x / R][0];
  __syncthreads();
  if (threadIdx.x < WARPS * R) {
    const int w = threadIdx.x / R, r = threadIdx.x - w * R;
    float top = sm[0][r];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) top = fmaxf(top, sm[i][r]);
    // (a warp without tiles has sums of zero; one whose scores are no numbers passes that on)
    const float e = sm[w][r] == -INFINITY ? 0.f : fast_exp2(sm[w][r] - top);
    ww[w][r] = e * back;
    sl[w][r] *= e;
  }
  __syncthreads();
  if (threadIdx.x < R) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) sum += sl[i][threadIdx.x];
    total[threadIdx.x] = sum;
  }
  __syncthreads();
  const bool single = pc.pieces == 1;
  float* po = a.po + (size_t)blockIdx.x * a.rows * HD;
  for (int i = threadIdx.x; i < nrows * HD; i += THREADS) {
    const int r = i / HD;
    float acc = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) acc += ww[w][r] * so[(size_t)w * R * HD + i];
    acc /= total[r];
    const size_t at = ((size_t)pc.b * a.nh + h0) * HD + i;
    if (!single) po[i] = acc;
    else if (a.out_f32) reinterpret_cast<float*>(a.out)[at] = acc;
    else reinterpret_cast<bf16*>(a.out)[at] = __float2bfloat16_rn(acc);
  }
  if (!single && threadIdx.x < nrows) {
    float top = sm[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) top = fmaxf(top, sm[i][threadIdx.x]);
    a.pml[(size_t)blockIdx.x * a.rows + threadIdx.x] = make_float2(top, total[threadIdx.x]);
  }
}

// A block a (request, chunk of heads, head): the pieces' results, weighted by their shares of the sum, in order.
constexpr int JOIN_THREADS = 256, JOIN_LANES = HD / 4, JOIN_GROUPS = JOIN_THREADS / JOIN_LANES;
__global__ void __launch_bounds__(JOIN_THREADS)
quant_join_kernel(const DecodeArgs a) {
  __shared__ float4 part[JOIN_GROUPS][JOIN_LANES];
  __shared__ float part_l[JOIN_GROUPS];
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, G = a.nh / a.nkv, heads = a.nkv * a.chunks;
  const int kvh = h / G, chunk = (h - kvh * G) / a.rows, r = h - kvh * G - chunk * a.rows;
  const int lane = threadIdx.x & 31;
  const int size = piece_size(a, lane);
  int before = 0, pieces = 1;
  for (int b0 = 0; b0 <= b; b0 += 32) {
    const int i = b0 + lane;
    int n = i <= b ? max(1, (request_tiles(a, request_length(a, i)) + size - 1) / size) : 0;
    pieces = __shfl_sync(0xffffffffu, n, b & 31);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    before += n;
  }
  if (pieces == 1) return;
  before -= pieces;
  const float2* ml = a.pml + ((size_t)before * heads + kvh * a.chunks + chunk) * a.rows + r;
  const float* po = a.po + (((size_t)before * heads + kvh * a.chunks + chunk) * a.rows + r) * HD;
  const size_t step = (size_t)heads * a.rows;
  float top = -INFINITY;
  for (int i = lane; i < pieces; i += 32) top = fmaxf(top, __ldcg(ml + i * step).x);
  top = warp_max(top);
  const int group = threadIdx.x / JOIN_LANES, c = threadIdx.x - group * JOIN_LANES;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = group; i < pieces && group < JOIN_GROUPS; i += JOIN_GROUPS) {
    const float2 x = __ldcg(ml + i * step);
    const float4 v = __ldcg(reinterpret_cast<const float4*>(po + i * step * HD) + c);
    const float w = (x.x == -INFINITY ? 0.f : fast_exp2(x.x - top)) * x.y;
    sum += w;
    acc.x += w * v.x, acc.y += w * v.y, acc.z += w * v.z, acc.w += w * v.w;
  }
  if (group < JOIN_GROUPS) part[group][c] = acc;          // (head sizes that do not divide the block)
  if (group < JOIN_GROUPS && c == 0) part_l[group] = sum;
  __syncthreads();
  if (group == 0) {
#pragma unroll
    for (int i = 1; i < JOIN_GROUPS; ++i) {
      const float4 v = part[i][c];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
      sum += part_l[i];
    }
    const float inv = 1.f / sum;
    const size_t at = ((size_t)b * a.nh + h) * HD + 4 * c;
    if (a.out_f32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at) =
          make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
      __nv_bfloat162* d = reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<bf16*>(a.out) + at);
      d[0] = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
      d[1] = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    }
  }
}

template <int NT, bool FP8, int PARTS, bool WHOLE, bool STEP>
int launch_decode(DecodeArgs a, int sms, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  constexpr auto kernel = quant_decode_kernel<NT, FP8, PARTS, WHOLE, STEP>;
  constexpr int smem = WARPS * 8 * NT * HD * 4;
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
  a.slots = sms * std::min(std::max(1, blocks_a_sm[dev]), kMostBlocks);
  const int heads = a.nkv * a.chunks, N = a.slots / heads;
  // the most pieces there can be (find_piece), and the most there are worth their while
  long long pieces = 2 * a.B <= N ? N + 1 : (2LL * a.slots + heads - 1) / heads + a.B;
  const long long keys = a.span ? std::min(std::abs((long long)a.span), (long long)a.limit) : a.limit;
  const long long tiles = (keys + TILE - 1) / TILE + 1;
  pieces = std::min(pieces, (long long)a.B * ((tiles + kLeastTiles - 1) / kLeastTiles));
  const long long blocks = std::max(pieces, (long long)a.B) * heads;
  if (blocks > 0x7fffffffLL) return -5;
  const bool joined = pieces > a.B;
  if (joined) {
    const size_t rows = (size_t)blocks * a.rows;
    if (scratch_bytes < rows * (HD + 2) * 4) return -7;
    a.po = (float*)scratch;
    a.pml = (float2*)((float*)scratch + rows * HD);
  }
  int e = launch_kernel(kernel, dim3((unsigned)blocks), dim3(THREADS), smem, stream, a);
  if (e || !joined) return e;
  return launch_kernel(quant_join_kernel, dim3(a.nh, a.B), dim3(JOIN_THREADS), 0, stream, a);
}

}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// Scratch that any call with these sizes is content with.
GF_EXPORT long long gf_quant_decode_scratch(int B, int nh, int nkv, int sms) {
  const int G = nh / nkv, chunks = (G + 15) / 16, rows = (G + chunks - 1) / chunks, heads = nkv * chunks;
  const long long slots = (long long)sms * kMostBlocks;
  return (2 * slots + (long long)(B + 2) * heads) * rows * (HD + 2) * 4;
}

// q [B, nh HD], or with `step` q | k | v [B, (nh + 2 nkv) HD] and the table of angles as gf_quant_write takes it.
GF_EXPORT int gf_quant_decode(const void* q, int q_stride, int q_f32, void* codes, int fp8, float* scales,
                              const int* block_table, int table_stride, int table_width, const int* lengths,
                              void* out, int out_f32, int B, int nh, int nkv, int page, int span, float scale,
                              int step, const float* table, int table_rows, int rot, int neighbours, int sms,
                              void* scratch, long long scratch_bytes, void* stream) {
  if (B <= 0) return B < 0 ? -3 : 0;
  if (nkv < 1 || nh < nkv || nh % nkv || page < 1 || table_width < 0 || B > 65535 || sms < 1) return -3;
  if (step && (rot < 0 || rot % 2 || rot > HD || (rot && (!table || table_rows < 1)))) return -3;
  DecodeArgs a = {};
  a.q = q, a.q_stride = q_stride, a.q_f32 = q_f32;
  a.codes = (uint8_t*)codes, a.scales = scales;
  a.block_table = block_table, a.table_stride = table_stride;
  a.limit = (int)min((long long)table_width * page, 0x7fffffe0LL);
  a.lengths = lengths, a.out = out, a.out_f32 = out_f32;
  a.B = B, a.nh = nh, a.nkv = nkv, a.page = page, a.span = span, a.scale = scale;
  a.page_shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1;
  a.table = table, a.table_rows = table_rows > 0 ? table_rows : 1, a.rot = rot, a.neighbours = neighbours;
  const int G = nh / nkv;
  a.chunks = (G + 15) / 16, a.rows = (G + a.chunks - 1) / a.chunks;
  const auto go = [&](auto nt, auto kind, auto parts, auto whole, auto fused) {
    return launch_decode<decltype(nt)::value, decltype(kind)::value, decltype(parts)::value, decltype(whole)::value,
                         decltype(fused)::value>(a, sms, scratch, (size_t)scratch_bytes, (cudaStream_t)stream);
  };
  const auto pick_bool = [](bool x, auto next) {
    return x ? next(std::true_type()) : next(std::false_type());
  };
  return pick_bool(fp8 != 0, [&](auto kind) {
    return pick_bool(page % TILE == 0, [&](auto whole) {
      return pick_bool(step != 0, [&](auto fused) {
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        if (q_f32) return a.rows > 8 ? go(Two(), kind, Two(), whole, fused) : go(One(), kind, Two(), whole, fused);
        return a.rows > 8 ? go(Two(), kind, One(), whole, fused) : go(One(), kind, One(), whole, fused);
      });
    });
  });
}
