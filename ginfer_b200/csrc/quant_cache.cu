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
// A row is held by LANES lanes of 8 channels each; a group of LANES lanes takes HU heads of one token, so
// that their loads are under way together and the angles of the token's position are read once for them.
template <typename T, int LANES, int HU>
__global__ void __launch_bounds__(256)
quant_write_kernel(const T* __restrict__ qkv, int row_stride, int tokens, int nh, int nkv, int hd,
                   const float* __restrict__ table, int table_rows, int rot, int neighbours,
                   const int* __restrict__ positions, const int* __restrict__ slots, T* __restrict__ q_out,
                   uint8_t* __restrict__ codes, int fp8, float* __restrict__ scales, int page, int num_slots,
                   int vec) {
  pdl_trigger();
  pdl_wait();
  const int heads = nh + 2 * nkv, sets = (heads + HU - 1) / HU;
  const int lane = threadIdx.x & (LANES - 1);
  const long long group = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / LANES;
  const int t = (int)(group / sets);
  const int h0 = (int)(group - (long long)t * sets) * HU;
  const bool here = t < tokens && lane * 8 < hd;
  const int c0 = lane * 8;
  const T* row = qkv + (size_t)(here ? t : 0) * row_stride;
  const int slot = t < tokens ? fresh_index(slots + t) : -1;
  const bool keep = slot >= 0 && slot < num_slots;

  float x[HU][8], y[HU][8];
  const int half = rot >> 1;
  // the channels that this lane's are paired with: its own where neighbours turn together
  const bool turns = here && c0 < rot;
  const int shift = c0 < half ? half : -half;
  // (halves that are no multiple of 8: a lane's 8 channels may have partners on both sides)
  const bool plain_pairs = !neighbours && (half & 7) == 0;
#pragma unroll
  for (int i = 0; i < HU; ++i) {
    const int h = h0 + i;
    if (here && h < heads) {
      load8(row + (size_t)h * hd + c0, x[i], vec);
      if (turns && h < nh + nkv && plain_pairs) load8(row + (size_t)h * hd + c0 + shift, y[i], vec);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
    }
  }
  if (turns && h0 < nh + nkv) {
    const int p = min(max(fresh_index(positions + t), 0), table_rows - 1);
    const float* cs = table + (size_t)p * rot;
    float c[8], s[8];
    if (neighbours) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = cs[(c0 >> 1) + e < half ? (c0 >> 1) + e : 0],
                                  s[e] = cs[(c0 >> 1) + e < half ? half + (c0 >> 1) + e : 0];
    } else if (plain_pairs) {
      const int j = c0 < half ? c0 : c0 - half;
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = cs[j + e], s[e] = cs[half + j + e];
    }
#pragma unroll
    for (int i = 0; i < HU; ++i) {
      const int h = h0 + i;
      if (h >= nh + nkv) continue;
      if (neighbours) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c0 + 2 * e < rot) turn_pair(x[i][2 * e], x[i][2 * e + 1], c[e], s[e]);
      } else if (plain_pairs) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[i][e] = c0 < half ? turned_first(x[i][e], y[i][e], c[e], s[e])
                              : turned_second(y[i][e], x[i][e], c[e], s[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int ch = c0 + e;
          if (ch >= rot) continue;
          const int j = ch < half ? ch : ch - half;
          const float o = to_f32(row[(size_t)h * hd + (ch < half ? ch + half : j)]);
          x[i][e] = ch < half ? turned_first(x[i][e], o, cs[j], cs[half + j])
                              : turned_second(o, x[i][e], cs[j], cs[half + j]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HU; ++i) {
    const int h = h0 + i;
    if (h < nh) {                          // a group's lanes agree on h: its shuffles below are whole
      if (here) store8(q_out + (size_t)t * nh * hd + (size_t)h * hd + c0, x[i]);
    }
    const bool kv = t < tokens && h >= nh && h < heads;
    const uint32_t top = group_max_bits<LANES>(kv ? max_bits8(x[i]) : 0u);
    if (kv && keep) {
      const int which = h >= nh + nkv, kvh = h - nh - which * nkv;
      const RowScale rs = row_scale(top, fp8);
      const int pg = slot / page, off = slot - pg * page;
      const size_t at = (size_t)pg * nkv + kvh;
      if (here)
        *reinterpret_cast<uint2*>(codes + ((at * 2 + which) * page + off) * hd + c0) =
            quantise8(x[i], rs, fp8);
      if (lane == 0) scales[(at * page + off) * 2 + which] = rs.scale;
    }
  }
}

template <typename T, int LANES>
int launch_write(const void* qkv, int row_stride, int tokens, int nh, int nkv, int hd, const float* table,
                 int table_rows, int rot, int neighbours, const int* positions, const int* slots, void* q_out,
                 uint8_t* codes, int fp8, float* scales, int page, int num_slots, int vec,
                 cudaStream_t stream) {
  const int heads = nh + 2 * nkv;
  const bool one = (long long)tokens * heads * LANES <= 148 * 1024;
  const int hu = one ? 1 : 4;
  const long long threads = (long long)tokens * ((heads + hu - 1) / hu) * LANES;
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) return -5;
  const auto run = [&](auto kernel) {
    return launch_kernel(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)qkv, row_stride,
                         tokens, nh, nkv, hd, table, table_rows, rot, neighbours, positions, slots, (T*)q_out,
                         codes, fp8, scales, page, num_slots, vec);
  };
  return one ? run(quant_write_kernel<T, LANES, 1>) : run(quant_write_kernel<T, LANES, 4>);
}

// -------------------------------------------------------------------------------------- read
// Dense [2, B, S, kv heads, hd]: position s of request b through its block table where first <= s < length,
// zeros elsewhere; or, with `slots`, row s of [2, 1, S, kv heads, hd] from slot slots[s] (negative: zeros).
template <typename T>
__global__ void __launch_bounds__(256)
quant_read_kernel(const uint8_t* __restrict__ codes, int fp8, const float* __restrict__ scales,
                  const int* __restrict__ block_table, int table_stride, const int* __restrict__ lengths,
                  const int* __restrict__ first, const int* __restrict__ slots, int num_slots, int S, int nkv,
                  int hd, int page, T* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y;
  const int chunks = hd / 16, per_token = 2 * nkv * chunks;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long long)S * per_token) return;
  const int s = (int)(i / per_token);
  int u = (int)(i - (long long)s * per_token);
  const int which = u / (nkv * chunks);
  u -= which * nkv * chunks;
  const int kvh = u / chunks, ch = u - kvh * chunks;
  int pg = -1, off = 0;
  if (slots) {
    const int slot = fresh_index(slots + s);
    if (slot >= 0 && slot < num_slots) pg = slot / page, off = slot - pg * page;
  } else if (s < fresh_index(lengths + b) && (!first || s >= fresh_index(first + b))) {
    const int lp = s / page;
    pg = fresh_index(block_table + (size_t)b * table_stride + lp), off = s - lp * page;
  }
  float v[16];
  if (pg >= 0) {
    const size_t at = (size_t)pg * nkv + kvh;
    const uint4 raw = *reinterpret_cast<const uint4*>(codes + ((at * 2 + which) * page + off) * hd + ch * 16);
    const float sc = scales[(at * page + off) * 2 + which];
    values16(raw, fp8, v);
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = __fmul_rn(v[e], sc);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = 0.f;
  }
  T* o = out + ((((size_t)which * gridDim.y + b) * S + s) * nkv + kvh) * hd + ch * 16;
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) lo[e] = v[e], hi[e] = v[8 + e];
  store8(o, lo);
  store8(o + 8, hi);
}

}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// qkv [T, >= (nh + 2 nkv) hd] with `row_stride`; table [table_rows, rot] fp32 (cosines, sines) or null with
// rot 0; q_out [T, nh hd].  A slot outside [0, num_slots) is not written, a position outside the table takes
// its nearest row.
GF_EXPORT int gf_quant_write(const void* qkv, int row_stride, int dtype, int tokens, int nh, int nkv, int hd,
                             const float* table, int table_rows, int rot, int neighbours, const int* positions,
                             const int* slots, void* q_out, void* codes, int fp8, float* scales, int page,
                             int num_slots, void* stream) {
  if (tokens <= 0) return tokens < 0 ? -3 : 0;
  if (hd % 16 || hd < 16 || hd > 256 || nh < 1 || nkv < 1 || page < 1 || rot < 0 || rot % 2 || rot > hd ||
      (rot && (!table || table_rows < 1)))
    return -3;
  const size_t es = dtype == GF_F32 ? 4 : 2;
  const int vec = ((size_t)qkv % 16 == 0 && (size_t)row_stride * es % 16 == 0) ? 1 : 0;
  const auto go = [&](auto tag) {
    using T = decltype(tag);
    const auto run = [&](auto launch) {
      return launch(qkv, row_stride, tokens, nh, nkv, hd, table, table_rows, rot, neighbours, positions, slots,
                    q_out, (uint8_t*)codes, fp8, scales, page, num_slots, vec, (cudaStream_t)stream);
    };
    if (hd <= 32) return run(launch_write<T, 4>);
    if (hd <= 64) return run(launch_write<T, 8>);
    if (hd <= 128) return run(launch_write<T, 16>);
    return run(launch_write<T, 32>);
  };
  return dtype == GF_F32 ? go(float()) : go(bf16());
}

// block_table, lengths (and first, may be null) of B requests, out [2, B, S, nkv, hd]; or slots [S] with B = 1.
GF_EXPORT int gf_quant_read(const void* codes, int fp8, const float* scales, const int* block_table,
                            int table_stride, const int* lengths, const int* first, const int* slots,
                            int num_slots, int B, int S, int nkv, int hd, int page, void* out, int dtype,
                            void* stream) {
  if (B <= 0 || S <= 0) return B < 0 || S < 0 ? -3 : 0;
  if (hd % 16 || hd < 16 || hd > 256 || nkv < 1 || page < 1 || B > 65535) return -3;
  const long long units = (long long)S * 2 * nkv * (hd / 16), blocks = (units + 255) / 256;
  if (blocks > 0x7fffffffLL) return -5;
  const dim3 grid((unsigned)blocks, (unsigned)B);
  const auto go = [&](auto tag) {
    using T = decltype(tag);
    return launch_kernel(quant_read_kernel<T>, grid, dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)codes,
                         fp8, scales, block_table, table_stride, lengths, first, slots, num_slots, S, nkv, hd,
                         page, (T*)out);
  };
  return dtype == GF_F32 ? go(float()) : go(bf16());
}
