// Verification of drafted tokens against the target's probabilities, from given random numbers.
// Request b has the rows c0 = cu[b] .. c1 - 1 of the target's logits; the token of row c0 + i + 1 is its i-th draft, held
// against row c0 + i.  With p = softmax(x / T) of a row and q the draft's (all of it on the draft without its logits), a draft
// d stays while u q(d) < p(d); the token behind the last that stays is the first j at which the running sum of
// w = max(p - q, 0) (w = p behind the last draft) reaches u times the whole, among those with w > 0.
// One block a request, everything in 64 bits.
#include "common.cuh"

namespace gf {

constexpr int kVerify = 512;

struct VerifyArgs {
  const void* logits;          // rows of `stride`
  const void* draft;           // rows of `draft_stride` beside the target's, or null
  const int* tokens;           // [R]
  const int* cu;               // [B + 1]
  const float* temperature;    // [B]
  const float* u;              // [R]
  int* accepted;               // [B]
  int* next;                   // [B]
  long long stride, draft_stride;
  int R, V, B;
};

__device__ double block_total(double v, double* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  double t = 0.;
  for (int w = 0; w < kVerify / 32; ++w) t += scratch[w];
  return t;
}
// The largest logit of a row and its first place; NaN never wins (place 0 when nothing does).
template <typename T> __device__ void row_best(const T* x, int V, float* best, int* place, float* sv, int* si) {
  float v = -INFINITY;
  int at = 0x7fffffff;
  for (int j = threadIdx.x; j < V; j += kVerify) {
    const float y = to_f32(x[j]);
    if (y > v) v = y, at = j;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (ov > v || (ov == v && oi < at)) v = ov, at = oi;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sv[threadIdx.x >> 5] = v, si[threadIdx.x >> 5] = at;
  __syncthreads();
  v = sv[0], at = si[0];
  for (int w = 1; w < kVerify / 32; ++w)
    if (sv[w] > v || (sv[w] == v && si[w] < at)) v = sv[w], at = si[w];
  *best = v, *place = at == 0x7fffffff ? 0 : at;
}
// A logit's weight before the division by the row's sum.
__device__ __forceinline__ double weight(float x, float best, double heat) {
  if (!(x > -INFINITY)) return 0.;
  if (best == INFINITY) return x == INFINITY ? 1. : 0.;
  return exp(((double)x - (double)best) / heat);
}

template <typename T> __global__ void __launch_bounds__(kVerify) verify_simple_kernel(const VerifyArgs a) {
  __shared__ double scratch[kVerify];
  __shared__ float sv[kVerify / 32];
  __shared__ int si[kVerify / 32];
  __shared__ int found;
  const int b = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const int c0 = min(max(fresh_index(a.cu + b), 0), a.R), c1 = min(max(fresh_index(a.cu + b + 1), c0), a.R);
  if (c1 <= c0) {
    if (threadIdx.x == 0) a.accepted[b] = 0, a.next[b] = -1;
    return;
  }
  const double heat = fresh(a.temperature + b);
  const bool greedy = !(heat > 0.);
  const int V = a.V;
  for (int row = c0; row < c1; ++row) {
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const bool last = row + 1 == c1;
    const int d = last ? -1 : fresh_index(a.tokens + row + 1);
    const bool real = d >= 0 && d < V;
    float best;
    int place;
    row_best(x, V, &best, &place, sv, si);
    if (greedy) {
      if (!last && d == place) continue;
      if (threadIdx.x == 0) a.accepted[b] = row - c0, a.next[b] = place;
      return;
    }
    double s = 0.;
    for (int j = threadIdx.x; j < V; j += kVerify) s += weight(to_f32(x[j]), best, heat);
    const double P = block_total(s, scratch);
    const T* y = nullptr;
    double Q = 1.;
    float dbest = 0.f;
    if (!last && a.draft) {
      y = static_cast<const T*>(a.draft) + row * a.draft_stride;
      int unused;
      row_best(y, V, &dbest, &unused, sv, si);
      s = 0.;
      for (int j = threadIdx.x; j < V; j += kVerify) s += weight(to_f32(y[j]), dbest, heat);
      Q = block_total(s, scratch);
    }
    if (!last && real && P > 0.) {
      const double p = weight(to_f32(x[d]), best, heat) / P;
      const double q = y ? (Q > 0. ? weight(to_f32(y[d]), dbest, heat) / Q : 0.) : 1.;
      if ((double)fresh(a.u + row) * q < p) continue;
    }
    // the token behind: chunk by chunk in order
    auto rest = [&](int j, bool whole) {
      const double p = P > 0. ? weight(to_f32(x[j]), best, heat) / P : 0.;
      if (whole || last) return p;
      if (!y) return j == d ? 0. : p;
      return fmax(p - (Q > 0. ? weight(to_f32(y[j]), dbest, heat) / Q : 0.), 0.);
    };
    const int each = (V + kVerify - 1) / kVerify, j0 = min(V, (int)threadIdx.x * each), j1 = min(V, j0 + each);
    int pick = -1;
    for (int whole = 0; whole < 2 && pick < 0; ++whole) {          // (nothing left of p - q: p itself)
      double mine = 0.;
      for (int j = j0; j < j1; ++j) mine += rest(j, whole);
      __syncthreads();
      scratch[threadIdx.x] = mine;
      if (threadIdx.x == 0) found = -1;
      __syncthreads();
      double before = 0., total = 0.;
      for (int i = 0; i < kVerify; ++i) {
        if (i == threadIdx.x) before = total;
        total += scratch[i];
      }
      if (!(total > 0.)) {
        __syncthreads();
        continue;
      }
      const double target = (double)fresh(a.u + c1 - 1) * total;
      if (mine > 0. && before + mine >= target && (before < target || before == 0.)) {
        double run = before;
        for (int j = j0; j < j1; ++j) {
          const double w = rest(j, whole);
          run += w;
          if (run >= target && w > 0.) {
            atomicMax(&found, 0x7fffffff - j);                     // (the first of them)
            break;
          }
        }
      }
      __syncthreads();
      pick = found < 0 ? -1 : 0x7fffffff - found;
      __syncthreads();
      if (pick < 0) break;
    }
    if (threadIdx.x == 0) a.accepted[b] = row - c0, a.next[b] = pick < 0 ? place : pick;
    return;
  }
}

}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

GF_EXPORT int gf_verify(const char* words) {
  const long long* w = reinterpret_cast<const long long*>(words);
  VerifyArgs a;
  int i = 0;
  auto ptr = [&] { return reinterpret_cast<void*>(w[i++]); };
  a.logits = ptr(), a.stride = w[i++];
  const int type = (int)w[i++];
  a.draft = ptr(), a.draft_stride = w[i++];
  a.tokens = (const int*)ptr(), a.cu = (const int*)ptr(), a.temperature = (const float*)ptr(), a.u = (const float*)ptr();
  a.accepted = (int*)ptr(), a.next = (int*)ptr();
  a.R = (int)w[i++], a.V = (int)w[i++], a.B = (int)w[i++];
  cudaStream_t stream = (cudaStream_t)ptr();
  if (a.B <= 0) return 0;
  return launch_kernel(type == GF_BF16 ? verify_simple_kernel<bf16> : verify_simple_kernel<float>, dim3(a.B),
                       dim3(kVerify), 0, stream, a);
}
