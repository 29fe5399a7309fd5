// Attention of a batch's newest tokens over a prefix that a group of requests shares and over their own tokens:
//   out[t, h] = sum_c softmax_c(scale <q[t, h], K_c>) V_c.
// One block a (request, head), a warp a key at a time, everything in 32 bits.
#include "shared_prefix.cuh"

namespace gf {

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

}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// `words`: q, its row stride and type, k, v, pages, page, prefix_table and its stride, prefix_lens, groups, prefix limit,
// table and its stride, lengths, requests, limit, cu_groups, cu, out, rows, heads, kv heads, head size, stream; then the
// scale as a double.
GF_EXPORT int gf_prefix_attend(const char* words) {
  const long long* w = reinterpret_cast<const long long*>(words);
  PrefixArgs a;
  int i = 0;
  auto ptr = [&] { return reinterpret_cast<void*>(w[i++]); };
  auto num = [&] { return (int)w[i++]; };
  a.q = ptr(), a.q_stride = num();
  const int type = num();
  a.k = ptr(), a.v = ptr(), a.pages = num(), a.page = num();
  a.prefix_table = (const int*)ptr(), a.prefix_stride = num(), a.prefix_lens = (const int*)ptr();
  a.G = num(), a.prefix_limit = num();
  a.table = (const int*)ptr(), a.table_stride = num(), a.lengths = (const int*)ptr(), a.B = num(), a.limit = num();
  a.cu_groups = (const int*)ptr(), a.cu = (const int*)ptr(), a.out = ptr();
  a.T = num(), a.nh = num(), a.nkv = num(), a.hd = num();
  cudaStream_t stream = (cudaStream_t)ptr();
  a.scale = (float)*reinterpret_cast<const double*>(w + i);
  if (a.B <= 0 || a.T <= 0) return 0;
  return launch_kernel(type == GF_BF16 ? prefix_simple_kernel<bf16> : prefix_simple_kernel<float>, dim3(a.B, a.nh),
                       dim3(32 * kWarps), 0, stream, a);
}
