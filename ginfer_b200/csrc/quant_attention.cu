// One new token's attention over a paged key-value cache of 8 bits (quant_cache.cu: its formulas and
// lay-out), compiled for one head size (-DGF_HEAD_DIM=<multiple of 16, at most 256>).
//
// For a request of `len` tokens the query is the last one, at position p = len - 1; it sees the keys
// first_visible_key(p, span) .. p.  out = sum_c softmax_c(scale <q, K_c>) V_c; a request without a
// token gives zeros.
#include "quant.cuh"

#ifndef GF_HEAD_DIM
#define GF_HEAD_DIM 128
#endif

namespace gf {

constexpr int HD = GF_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16, <= 256");
constexpr float kLog2E = 1.4426950408889634f;

// A block of four warps a (request, query head); a warp takes every fourth key, a lane HD/32 of its channels.
template <typename TQ, typename TO>
__global__ void __launch_bounds__(128)
quant_decode_kernel(const TQ* __restrict__ q, int q_stride, const uint8_t* __restrict__ codes, int fp8,
                    const float* __restrict__ scales, const int* __restrict__ block_table, int table_stride,
                    int table_width, const int* __restrict__ lengths, TO* __restrict__ out, int nh, int nkv,
                    int page, int span, float scale) {
  constexpr int N = (HD + 31) / 32;
  __shared__ float so[4][HD], sm[4], sl[4];
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / (nh / nkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = (int)min((long long)fresh_index(lengths + b), (long long)table_width * page);
  const int lo = len > 0 ? first_visible_key(len - 1, span) : 0;
  float qv[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    o[i] = 0.f;
    qv[i] = i * 32 + lane < HD ? fresh(q + (size_t)b * q_stride + (size_t)h * HD + i * 32 + lane) : 0.f;
  }
  for (int c = lo + warp; c < len; c += 4) {
    const int lp = c / page, off = c - lp * page;
    const size_t at = (size_t)fresh_index(block_table + (size_t)b * table_stride + lp) * nkv + kvh;
    const uint8_t* k = codes + (at * 2 * page + off) * HD;
    const uint8_t* v = k + (size_t)page * HD;
    const float2 sc = __ldcg(reinterpret_cast<const float2*>(scales) + at * page + off);
    float dot = 0.f, vv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      vv[i] = 0.f;
      if (i * 32 + lane < HD) {
        float four[4];
        values4(__ldcg(k + i * 32 + lane), fp8, four);
        dot = fmaf(qv[i], four[0], dot);
        values4(__ldcg(v + i * 32 + lane), fp8, four);
        vv[i] = four[0];
      }
    }
    const float s = warp_sum(dot) * sc.x * scale;
    const float mn = fmaxf(m, s);
    // (a score that is no number makes the row none: exp2f hands it on)
    const float corr = exp2f((m - mn) * kLog2E), p = exp2f((s - mn) * kLog2E);
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = fmaf(p * sc.y, vv[i], o[i] * corr);
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * 32 + lane < HD) so[warp][i * 32 + lane] = o[i];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float w[4], total = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = sm[i] == -INFINITY ? 0.f : exp2f((sm[i] - mm) * kLog2E);
    total += w[i] * sl[i];
  }
  for (int d = threadIdx.x; d < HD; d += 128) {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc += w[i] * so[i][d];
    out[((size_t)b * nh + h) * HD + d] = from_f32<TO>(lo < len ? acc / total : 0.f);
  }
}

}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

GF_EXPORT int gf_quant_decode(const void* q, int q_stride, int q_dtype, const void* codes, int fp8,
                              const float* scales, const int* block_table, int table_stride, int table_width,
                              const int* lengths, void* out, int out_dtype, int B, int nh, int nkv, int page,
                              int span, float scale, void* stream) {
  if (B <= 0) return B < 0 ? -3 : 0;
  if (nkv < 1 || nh < nkv || nh % nkv || page < 1 || table_width < 0 || B > 65535) return -3;
  const auto run = [&](auto tq, auto to) {
    using TQ = decltype(tq);
    using TO = decltype(to);
    return launch_kernel(quant_decode_kernel<TQ, TO>, dim3(nh, B), dim3(128), 0, (cudaStream_t)stream,
                         (const TQ*)q, q_stride, (const uint8_t*)codes, fp8, scales, block_table, table_stride,
                         table_width, lengths, (TO*)out, nh, nkv, page, span, scale);
  };
  if (q_dtype == GF_F32) return out_dtype == GF_F32 ? run(float(), float()) : run(float(), bf16());
  return out_dtype == GF_F32 ? run(bf16(), float()) : run(bf16(), bf16());
}
