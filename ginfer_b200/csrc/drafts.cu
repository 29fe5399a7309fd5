// Verification of drafted tokens against the target's probabilities, from given random numbers.
// Request b has the rows c0 = cu[b] .. c1 - 1 of the target's logits; the token of row c0 + i + 1 is its i-th draft, held
// against row c0 + i.  With p = softmax(x / T) of a row and q the draft's (all of it on the draft without its logits), a draft
// d stays while u q(d) < p(d); the token behind the last that stays is the first j at which the running sum of
// w = max(p - q, 0) (w = p behind the last draft) reaches u times the whole, among those with w > 0.
//
// What bounds it is reading the logits, once.  Two launches:
//  * verify_scan_kernel: every row in pieces of kPiece logits, each leaves its maximum and, relative to that, the sum of its
//    weights in 32 bits (requests of temperature zero: the maximum's first place).
//  * verify_decide_kernel: a cluster of blocks a request adds the pieces up, goes through the drafts and draws the next token
//    from the one row that it needs.
// 32 bits are enough to decide on nearly every draft; where u q(d) and p(d) are within kMargin of one another, the two rows'
// sums are taken again in 64 bits.  The drawn token is met by errors of the order of 2^-24 now and then (a border between two
// tokens is as near as 1 / V), so that everything about it is in 64 bits: weights above e^-20 of the largest, and all sums;
// a smaller weight's own error in 32 bits, 2^-22 of it, is below 2^-50 of the whole.
#include "common.cuh"
#include "tc_common.cuh"

namespace gf {
namespace {

constexpr int kScan = 256, kEach = 16, kPiece = kScan * kEach;        // threads of a scanning block, logits of a thread
constexpr int kDecide = 512, kWarps = kDecide / 32, kBatch = 32;      // rows whose sums are at hand at a time
constexpr int kMostCluster = 8;
// Relative error that the 32-bit sums may have: exponents are off by 2^-23 of up to 20 and the exponential by 2^-22, sums of
// 16 and across threads by less: 4e-6 for p and for q; ten times that.
constexpr double kMargin = 8e-5;
constexpr float kLog2E = 1.4426950408889634f;

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
  int R, V, B, pieces;
  float2* part;                // [R][2][pieces]: (maximum, sum), or (maximum, its place's bits) of the target's, the draft's row
};

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
// A row in groups of 16 bytes that start at multiples of 16: group g has the logits g * kVec - mis on.
template <typename T> struct Row {
  const T* x;
  int mis, V;
  __device__ __forceinline__ Row(const void* base, long long stride, int row, int V_)
      : x(static_cast<const T*>(base) + row * stride), V(V_) {
    mis = (int)(((size_t)x / sizeof(T)) % kVec<T>);
  }
  __device__ __forceinline__ int groups() const { return (V + mis + kVec<T> - 1) / kVec<T>; }
  __device__ __forceinline__ float at(int j) const {
    const float y = j >= 0 && j < V ? fresh(x + j) : -INFINITY;
    return y == y ? y : -INFINITY;                    // (a NaN counts as nothing)
  }
  // Group g's logits, -inf outside the row.
  __device__ __forceinline__ void load(int g, float (&v)[kVec<T>]) const {
    const int j = g * kVec<T> - mis;
    if (j >= 0 && j + kVec<T> <= V) {
      const uint4 raw = __ldcg(reinterpret_cast<const uint4*>(x + j));
      if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y);
        v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
      } else {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[i] = v[i] == v[i] ? v[i] : -INFINITY;
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[i] = at(j + i);
    }
  }
};

struct Span {
  int first, end;
};
__device__ __forceinline__ Span rows_of(const VerifyArgs& a, int b) {
  const int c0 = min(max(fresh_index(a.cu + b), 0), a.R), c1 = min(max(fresh_index(a.cu + b + 1), 0), a.R);
  return {c0, max(c0, c1)};
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2(e) / T, finite: times a difference of zero it is zero
__device__ __forceinline__ float inverse_heat(float heat) { return fminf(kLog2E / heat, 1e30f); }
// A logit's weight beside the row's largest one, in 32 bits.
__device__ __forceinline__ float weight32(float x, float best, float c) {
  if (x == best) return 1.f;                          // (infinities among them)
  return x == -INFINITY || best == INFINITY ? 0.f : fast_exp2((x - best) * c);
}

// ------------------------------------------------------------------------------------- rows in pieces
template <typename T>
__global__ void __launch_bounds__(kScan) verify_scan_kernel(const VerifyArgs a) {
  __shared__ float2 part[kScan / 32];
  const int b = blockIdx.x, piece = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int G = kEach / kVec<T>;                  // groups of a thread
  pdl_trigger();
  pdl_wait();
  const Span rows = rows_of(a, b);
  const float heat = fresh(a.temperature + b);
  const bool greedy = !(heat > 0.f);
  const float c = inverse_heat(heat);
  for (int row = rows.first + blockIdx.z; row < rows.end; row += gridDim.z) {
    for (int which = 0; which < (a.draft && !greedy && row + 1 < rows.end ? 2 : 1); ++which) {
      const Row<T> x(which ? a.draft : a.logits, which ? a.draft_stride : a.stride, row, a.V);
      float v[G][kVec<T>], top = -INFINITY;
      const int g0 = piece * (kPiece / kVec<T>) + threadIdx.x, end = x.groups();
#pragma unroll
      for (int i = 0; i < G; ++i) {
        if (g0 + i * kScan < end) {
          x.load(g0 + i * kScan, v[i]);
        } else {
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) v[i][k] = -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) top = fmaxf(top, v[i][k]);
      top = warp_max(top);
      float second = 0.f;
      if (greedy) {
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k)
            if (v[i][k] == top) at = min(at, (g0 + i * kScan) * kVec<T> - x.mis + k);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
        second = __int_as_float(at);
      } else if (top > -INFINITY) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
          for (int k = 0; k < kVec<T>; k += 2) s0 += weight32(v[i][k], top, c), s1 += weight32(v[i][k + 1], top, c);
        second = warp_sum(s0 + s1);
      }
      __syncthreads();
      if (lane == 0) part[warp] = make_float2(top, second);
      __syncthreads();
      if (threadIdx.x == 0) {
        float2 y = part[0];
        for (int w = 1; w < kScan / 32; ++w) {
          const float2 z = part[w];
          if (greedy) {
            if (z.x > y.x || (z.x == y.x && __float_as_int(z.y) < __float_as_int(y.y))) y = z;
          } else if (z.x > -INFINITY) {
            const float best = fmaxf(y.x, z.x);
            y.y = y.y * weight32(y.x, best, c) + z.y * weight32(z.x, best, c);
            y.x = best;
          }
        }
        a.part[((size_t)row * 2 + which) * a.pieces + piece] = y;
      }
    }
  }
}

// ------------------------------------------------------------------------------------- decisions
// A logit's weight beside the row's largest one: in 64 bits where it counts (see above).
struct Heat {
  double inv;                  // 1 / T
  float c;
};
__device__ __forceinline__ double weight64(float x, float best, const Heat& h) {
  if (x == best) return x == -INFINITY ? 0. : 1.;
  if (x == -INFINITY || best == INFINITY) return 0.;
  const float e = (x - best) * h.c;
  if (e < -29.f) return (double)fast_exp2(e);         // (2^-29 is e^-20)
  return exp(((double)x - (double)best) * h.inv);
}
__device__ __forceinline__ double shfl_xor(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// What a row's weights are relative to, and their sum.
struct Total {
  float best;
  double sum;
};
struct Cluster {
  uint32_t rank, size;
  int round;
  double (*slots)[2];          // [2][2] of this block
  // Both numbers' sums over the cluster's blocks, in the order of their ranks; `before`: what the blocks ahead of this one have of the
  // first.  By all threads; `mine` is the block's, known to thread 0.
  __device__ __forceinline__ void add(double mine0, double mine1, double& all0, double& all1, double& before) {
    double* at = slots[round & 1];
    if (threadIdx.x == 0) at[0] = mine0, at[1] = mine1;
    cluster_sync();
    all0 = all1 = before = 0.;
    for (uint32_t r = 0; r < size; ++r) {
      const uint32_t from = dsmem_addr(smem_u32(at), r);
      double x, y;
      asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(x), "=d"(y) : "r"(from) : "memory");
      if (r == rank) before = all0;
      all0 += x, all1 += y;
    }
    ++round;                   // (two slots in turn: nobody writes one before all have read it)
  }
};

template <typename T>
__global__ void __launch_bounds__(kDecide) verify_decide_kernel(const VerifyArgs a) {
  __shared__ Total totals[kBatch][2];                 // of the batch's rows: the target's, the draft's
  __shared__ int places[kBatch];                      // greedy: the arg-max
  __shared__ double sums[kWarps][2];
  __shared__ __align__(16) double slots[2][2];
  __shared__ int verdict[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Cluster cl{cluster_rank(), 0, 0, slots};
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cl.size));
  const int b = blockIdx.x / cl.size;
  pdl_trigger();
  pdl_wait();
  const Span rows = rows_of(a, b);
  const int n = rows.end - rows.first;
  if (n == 0) {                                       // (the whole cluster)
    if (cl.rank == 0 && threadIdx.x == 0) a.accepted[b] = 0, a.next[b] = -1;
    return;
  }
  const float heat = fresh(a.temperature + b);
  const bool greedy = !(heat > 0.f);
  const Heat h{1. / (double)heat, inverse_heat(heat)};
  // this block's share of a row's groups of 16 bytes, and the warp's of that, in order
  auto share_of = [&](int groups, int& w0, int& w1) {
    const int each = (groups + (int)cl.size - 1) / (int)cl.size, g0 = min(groups, (int)cl.rank * each), g1 = min(groups, g0 + each);
    const int per = (g1 - g0 + kWarps - 1) / kWarps;
    w0 = min(g1, g0 + warp * per), w1 = min(g1, w0 + per);
  };
  // both rows' sums of weights in 64 bits
  auto exact_totals = [&](int row, bool with_draft, float best, float draft_best, double& P, double& Q) {
    double s[2] = {0., 0.};
    for (int which = 0; which < (with_draft ? 2 : 1); ++which) {
      const Row<T> x(which ? a.draft : a.logits, which ? a.draft_stride : a.stride, row, a.V);
      const float top = which ? draft_best : best;
      int w0, w1;
      share_of(x.groups(), w0, w1);
      for (int g = w0 + lane; g < w1; g += 32) {
        float v[kVec<T>];
        x.load(g, v);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) s[which] += weight64(v[k], top, h);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[0] += shfl_xor(s[0], o), s[1] += shfl_xor(s[1], o);
    __syncthreads();
    if (lane == 0) sums[warp][0] = s[0], sums[warp][1] = s[1];
    __syncthreads();
    double m0 = 0., m1 = 0., unused;
    if (threadIdx.x == 0)
      for (int w = 0; w < kWarps; ++w) m0 += sums[w][0], m1 += sums[w][1];
    cl.add(m0, m1, P, Q, unused);
  };

  int stop = n - 1, in_batch = 0;
  bool refused = false, exact = false;
  double P = 0., Q = 0.;
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    // the batch's totals, a warp a row
    const int here = min(kBatch, n - i0);
    __syncthreads();
    for (int k = warp; k < 2 * here; k += kWarps) {
      const int i = k >> 1, which = k & 1, row = rows.first + i0 + i;
      if (which && (!a.draft || greedy || i0 + i == n - 1)) continue;
      const float2* part = a.part + ((size_t)row * 2 + which) * a.pieces;
      float best = -INFINITY;
      int at = 0x7fffffff;
      for (int q = lane; q < a.pieces; q += 32) {
        const float2 y = __ldcg(part + q);
        if (greedy && (y.x > best || (y.x == best && __float_as_int(y.y) < at))) at = __float_as_int(y.y);
        best = fmaxf(best, y.x);
      }
      double sum = 0.;
      if (greedy) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float ob = __shfl_xor_sync(0xffffffffu, best, o);
          const int oa = __shfl_xor_sync(0xffffffffu, at, o);
          if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
        }
      } else {
        best = warp_max(best);
        for (int q = lane; q < a.pieces; q += 32) {
          const float2 y = __ldcg(part + q);
          sum += (double)y.y * weight64(y.x, best, h);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor(sum, o);
      }
      if (lane == 0) {
        totals[i][which] = {best, sum};
        if (!which) places[i] = best == -INFINITY || at == 0x7fffffff ? 0 : at;
      }
    }
    __syncthreads();
    // the first row of the batch at which it ends: 0 the draft stays, 1 it does not, 2 the sums have to be taken again, 3 the last row
    int from = 0;
    bool done = false;
    while (true) {
      if (warp == 0) {
        int what = 0;
        const int i = lane, row = rows.first + i0 + i;
        if (i >= from && i < here) {
          if (i0 + i == n - 1) {
            what = 3;
          } else {
            const int d = fresh_index(a.tokens + row + 1);
            if (greedy) {
              what = d == places[i] ? 0 : 1;
            } else if (d < 0 || d >= a.V || !(totals[i][0].sum > 0.)) {
              what = 1;
            } else {
              const float xd = Row<T>(a.logits, a.stride, row, a.V).at(d);
              const double p = weight64(xd, totals[i][0].best, h) / totals[i][0].sum;
              double q = 1.;
              if (a.draft) {
                const float yd = Row<T>(a.draft, a.draft_stride, row, a.V).at(d);
                q = totals[i][1].sum > 0. ? weight64(yd, totals[i][1].best, h) / totals[i][1].sum : 0.;
              }
              const double left = (double)fresh(a.u + row) * q;
              what = left < p ? 0 : 1;
              if (fabs(left - p) <= kMargin * fmax(left, p) && p > 0.) what = 2;
            }
          }
        }
        const unsigned ends = __ballot_sync(0xffffffffu, what != 0);
        const int who = ends ? __ffs(ends) - 1 : -1;
        what = __shfl_sync(0xffffffffu, what, max(who, 0));
        if (lane == 0) verdict[0] = who, verdict[1] = what;
      }
      __syncthreads();
      const int who = verdict[0], what = verdict[1];
      __syncthreads();
      if (who < 0) break;                             // (all of the batch's drafts stay)
      in_batch = who, stop = i0 + who;
      exact = false;
      if (what == 2) {
        const int row = rows.first + stop;
        exact_totals(row, a.draft != nullptr, totals[who][0].best, totals[who][1].best, P, Q);
        exact = true;
        const int d = fresh_index(a.tokens + row + 1);
        const double p = weight64(Row<T>(a.logits, a.stride, row, a.V).at(d), totals[who][0].best, h) / P;
        double q = 1.;
        if (a.draft)
          q = Q > 0. ? weight64(Row<T>(a.draft, a.draft_stride, row, a.V).at(d), totals[who][1].best, h) / Q : 0.;
        if ((double)fresh(a.u + row) * q < p) {
          from = who + 1;
          continue;
        }
      }
      refused = what != 3;
      done = true;
      break;
    }
    if (done) break;
  }
  const int row = rows.first + stop;
  if (greedy) {
    if (cl.rank == 0 && threadIdx.x == 0) a.accepted[b] = stop, a.next[b] = places[in_batch];
    return;
  }
  // ---- the token behind the last draft that stays
  const bool with_draft = refused && a.draft;
  const float best = totals[in_batch][0].best, draft_best = with_draft ? totals[in_batch][1].best : 0.f;
  if (!exact) exact_totals(row, with_draft, best, draft_best, P, Q);
  const Row<T> x(a.logits, a.stride, row, a.V), y(with_draft ? a.draft : a.logits, with_draft ? a.draft_stride : a.stride, row, a.V);
  const int d = refused ? fresh_index(a.tokens + row + 1) : -1;
  const double inv_p = P > 0. ? 1. / P : 0., inv_q = with_draft && Q > 0. ? 1. / Q : 0.;
  int w0, w1;
  share_of(x.groups(), w0, w1);
  // a group's weights: without `whole` what p has more than q
  auto rest = [&](int g, bool whole, double (&w)[kVec<T>]) {
    float v[kVec<T>], z[kVec<T>];
    x.load(g, v);
    const int j = g * kVec<T> - x.mis;
    if (with_draft && !whole) {
      if (y.mis == x.mis) {
        y.load(g, z);
      } else {
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) z[k] = y.at(j + k);
      }
    }
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) {
      w[k] = weight64(v[k], best, h) * inv_p;
      if (with_draft && !whole) w[k] = fmax(w[k] - weight64(z[k], draft_best, h) * inv_q, 0.);
      else if (refused && !whole && j + k == d) w[k] = 0.;
    }
  };
  const double u = fmin(fmax((double)fresh(a.u + rows.end - 1), 0.), 1. - 0x1p-24);     // (whatever is handed in)
  for (int whole = 0; whole < 2; ++whole) {           // (where nothing is left of p - q: p itself)
    double mine = 0.;
    for (int g = w0 + lane; g < w1; g += 32) {
      double w[kVec<T>];
      rest(g, whole, w);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) mine += w[k];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += shfl_xor(mine, o);
    __syncthreads();
    if (lane == 0) sums[warp][0] = mine;
    __syncthreads();
    double block = 0., total, unused, before;
    for (int w = 0; w < kWarps; ++w) block += sums[w][0];
    cl.add(block, 0., total, unused, before);
    if (!(total > 0.)) continue;
    const double target = u * total;
    // the block, and in it the warp, in whose share the sum is reached (its last one, should rounding leave it short)
    const bool own = block > 0. && (before < target || before == 0.) && (before + block >= target || before + block == total);
    if (own) {
      double ahead = before;
      int owner = -1;
      double owner_ahead = 0.;
      for (int w = 0; w < kWarps; ++w) {
        if (sums[w][0] > 0.) {
          if (owner < 0 || ahead < target) owner = w, owner_ahead = ahead;
        }
        ahead += sums[w][0];
      }
      if (warp == owner) {
        double run = owner_ahead;
        int last = -1;
        bool found = false;
        for (int g = w0; g < w1 && !found; g += 32) {
          double w[kVec<T>], part = 0.;
          if (g + lane < w1) rest(g + lane, whole, w);
          else
#pragma unroll
            for (int k = 0; k < kVec<T>; ++k) w[k] = 0.;
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) part += w[k];
          double upto = part;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += up;
          }
          double at = run + (upto - part);
          int pick = -1, latest = -1;
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) {
            at += w[k];
            if (w[k] > 0.) {
              latest = (g + lane) * kVec<T> - x.mis + k;
              if (pick < 0 && at >= target) pick = latest;
            }
          }
          const unsigned hits = __ballot_sync(0xffffffffu, pick >= 0), some = __ballot_sync(0xffffffffu, latest >= 0);
          if (hits) last = __shfl_sync(0xffffffffu, pick, __ffs(hits) - 1), found = true;
          else if (some) last = __shfl_sync(0xffffffffu, latest, 31 - __clz(some));
          run += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) a.accepted[b] = stop, a.next[b] = last;
      }
    }
    cluster_sync();            // (nobody leaves while another reads its sums)
    return;
  }
  if (cl.rank == 0 && threadIdx.x == 0) a.accepted[b] = stop, a.next[b] = 0;      // (a row without a number)
  cluster_sync();
}

}  // namespace
}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// `words`: logits, row stride, type, the drafter's logits, their row stride, tokens, cu, temperature, u, accepted, next, rows,
// vocabulary, requests, scratch and its bytes, stream.
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
  a.part = (float2*)ptr();
  const long long room = w[i++];
  cudaStream_t stream = (cudaStream_t)ptr();
  if (a.B <= 0) return 0;
  const bool half = type == GF_BF16;
  a.pieces = (a.V + (half ? kVec<bf16> : kVec<float>) - 1 + kPiece - 1) / kPiece;
  if ((long long)a.R * 2 * a.pieces * 8 > room) return -5;
  if (a.pieces > 65535) return -6;
  const int z = a.R > a.B ? (a.R + a.B - 1) / a.B : 1;
  int rc = 0;
  if (a.R > 0)
    rc = launch_kernel(half ? verify_scan_kernel<bf16> : verify_scan_kernel<float>, dim3(a.B, a.pieces, z < 64 ? z : 64),
                       dim3(kScan), 0, stream, a);
  if (rc) return rc;
  return launch_kernel_cluster_dims(half ? verify_decide_kernel<bf16> : verify_decide_kernel<float>, dim3(a.B * kMostCluster),
                                    dim3(kDecide), 0, stream, kMostCluster, true, a);
}
