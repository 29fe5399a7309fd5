// Verification of drafted tokens against the target's probabilities, from given random numbers.
// Request b has the rows c0 = cu[b] .. c1 - 1 of the target's logits; the token of row c0 + i + 1 is its i-th draft, held
// against row c0 + i.  With p = softmax(x / T) of a row and q the draft's (all of it on the draft without its logits), a draft
// d stays while u q(d) < p(d); the token behind the last that stays is the first j at which the running sum of
// w = max(p - q, 0) (w = p behind the last draft) reaches u times the whole, among those with w > 0.
//
// What bounds it is reading the logits, once.  Two launches:
//  * verify_scan_kernel: every row in pieces, each leaves its maximum and, relative to that, the sum of its weights in 32 bits
//    (requests of temperature zero: the maximum's first place).
//  * verify_decide_kernel: a cluster of blocks a request adds the pieces up, goes through the drafts and draws the next token
//    from the one row that it needs.
// 32 bits are enough to decide on nearly every draft; where u q(d) and p(d) are within kMargin of one another, the two rows'
// sums are taken again in 64 bits.  The drawn token is met by errors of the order of 2^-24 now and then (there are V borders
// between tokens), so that its sums are in 64 bits, and so are the weights above e^-10 of the largest, of which there are
// few in a row that a model is sure about.  A smaller weight's factors 2^(n/256) come from a table in 64 bits and what is left,
// 1 + 1.4e-3 at most, from a short series in 32: off by 2e-10 of it, below 1e-14 of the largest.
#include <cstdlib>

#include "common.cuh"
#include "tc_common.cuh"

namespace gf {
namespace {

constexpr int kPiece = 1024;                            // logits of a piece
constexpr int kScan = 256, kScanBlocks = 2;             // threads of a scanning block, blocks an SM
constexpr int kSearch = 1024;                           // requests whose first rows a scanning block keeps
constexpr int kDecide = 512, kWarps = kDecide / 32, kBatch = 32;      // rows whose sums are at hand at a time
constexpr int kAhead = 4;                               // loads of a row that are under way
// Relative error that the 32-bit sums may have: exponents are off by 2^-23 of up to 20 and the exponential by 2^-22, sums of
// 64 and across lanes by less: 5e-6 for p and for q; eight times that for both.
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
template <typename T> constexpr int kLoads = kPiece / (32 * kVec<T>);              // a lane's of a piece
template <typename T> __device__ __forceinline__ void unpack(const uint4& raw, float (&v)[kVec<T>]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
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
  __device__ __forceinline__ bool whole(int g) const {
    const int j = g * kVec<T> - mis;
    return j >= 0 && j + kVec<T> <= V;
  }
  __device__ __forceinline__ uint4 raw(int g) const { return __ldcg(reinterpret_cast<const uint4*>(x + (g * kVec<T> - mis))); }
  // Group g's logits, -inf outside the row and for a NaN.
  __device__ __forceinline__ void load(int g, float (&v)[kVec<T>]) const {
    if (whole(g)) {
      unpack<T>(raw(g), v);
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[i] = fmaxf(v[i], -INFINITY);
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[i] = at(g * kVec<T> - mis + i);
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
// Two fp32 operations in one instruction: the operands are pairs in 64-bit registers.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// log2(e) / T, finite: times a difference of zero it is zero
__device__ __forceinline__ float inverse_heat(float heat) { return fminf(kLog2E / heat, 1e30f); }
// A logit's weight beside the row's largest one, in 32 bits.
__device__ __forceinline__ float weight32(float x, float best, float c) {
  if (x == best) return 1.f;                          // (infinities among them)
  return x == -INFINITY || best == INFINITY ? 0.f : fast_exp2((x - best) * c);
}

// ------------------------------------------------------------------------------------- rows in pieces
// A warp takes a piece after the other, the loads of the next one under way while it works on one.
template <typename T>
__global__ void __launch_bounds__(kScan, kScanBlocks) verify_scan_kernel(const VerifyArgs a) {
  __shared__ int starts[kSearch + 1];
  constexpr int GROUPS = 32 * kLoads<T>;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  const bool kept = a.B <= kSearch;
  if (kept)
    for (int i = threadIdx.x; i <= a.B; i += kScan) starts[i] = fresh_index(a.cu + i);
  __syncthreads();
  auto start_of = [&](int b) { return kept ? starts[b] : fresh_index(a.cu + b); };
  // pieces of the target's rows, then of the drafter's; this warp's are `me`, `me` + `all`, ...
  const long long half = (long long)a.R * a.pieces, units = a.draft ? 2 * half : half;
  const long long me = (long long)blockIdx.x * (kScan / 32) + (threadIdx.x >> 5), all = (long long)gridDim.x * (kScan / 32);
  for (long long u0 = me; u0 < units; u0 += 32 * all) {
    // the next 32 of them, a lane each: row, piece and temperature, if somebody asks for it
    const long long u = u0 + lane * all;
    const int my_which = u >= half;
    int my_row = 0, my_piece = 0;
    float my_heat = 0.f;
    bool there = u < units;
    if (there) {
      const long long at = my_which ? u - half : u;
      my_row = at >> 32 ? (int)(at / a.pieces) : (int)((unsigned)at / (unsigned)a.pieces);
      my_piece = (int)(at - (long long)my_row * a.pieces);
      int low = 0, high = a.B;                          // the last request that does not start behind the row
      while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (start_of(mid) <= my_row) low = mid;
        else high = mid;
      }
      const int end = start_of(low + 1);
      my_heat = fresh(a.temperature + low);
      there = my_row >= start_of(low) && my_row < end && !(my_which && (!(my_heat > 0.f) || my_row + 1 >= min(end, a.R)));
    }
    unsigned left = __ballot_sync(0xffffffffu, there);
    struct Unit {
      int row, which, piece;
      float heat;
      bool whole;
    };
    auto fetch = [&](uint4 (&raw)[kLoads<T>]) {            // the next of the ballot's
      const int who = __ffs(left) - 1;
      left &= left - 1;
      Unit x{__shfl_sync(0xffffffffu, my_row, who), __shfl_sync(0xffffffffu, my_which, who),
             __shfl_sync(0xffffffffu, my_piece, who), __shfl_sync(0xffffffffu, my_heat, who), false};
      const Row<T> r(x.which ? a.draft : a.logits, x.which ? a.draft_stride : a.stride, x.row, a.V);
      x.whole = r.whole(x.piece * GROUPS) && r.whole(x.piece * GROUPS + GROUPS - 1);
      if (x.whole) {
#pragma unroll
        for (int i = 0; i < kLoads<T>; ++i) raw[i] = r.raw(x.piece * GROUPS + i * 32 + lane);
      }
      return x;
    };
    auto work = [&](const Unit& x, const uint4 (&raw)[kLoads<T>]) {
      const Row<T> r(x.which ? a.draft : a.logits, x.which ? a.draft_stride : a.stride, x.row, a.V);
      const bool greedy = !(x.heat > 0.f);
      const float c = inverse_heat(x.heat);
      const int g0 = x.piece * GROUPS + lane;
      float top = -INFINITY, second = 0.f;
      if (x.whole) {
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kLoads<T>; ++i) {
          float v[kVec<T>];
          unpack<T>(raw[i], v);
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) t[k & 3] = fmaxf(t[k & 3], v[k]);       // (a NaN never is)
        }
        top = warp_max(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
        if (greedy) {
          int at = 0x7fffffff;
#pragma unroll
          for (int i = kLoads<T> - 1; i >= 0; --i) {
            float v[kVec<T>];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int k = kVec<T> - 1; k >= 0; --k)
              if (v[k] == top) at = (g0 + i * 32) * kVec<T> - r.mis + k;            // (the first of the lane's)
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
          second = __int_as_float(at);
        } else {
          // weights as they come; where one is no number (a NaN, infinities, a temperature of infinity) again with care
          const uint64_t c2 = pack2(c, c), m2 = pack2(-top, -top);
          uint64_t s2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
          for (int i = 0; i < kLoads<T>; ++i) {
            float v[kVec<T>];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int k = 0; k < kVec<T>; k += 2) {
              float e0, e1;
              unpack2(mul2(add2(pack2(v[k], v[k + 1]), m2), c2), e0, e1);
              s2[(k >> 1) & 1] = add2(s2[(k >> 1) & 1], pack2(fast_exp2(e0), fast_exp2(e1)));
            }
          }
          float s0, s1, s3, s4;
          unpack2(s2[0], s0, s1);
          unpack2(s2[1], s3, s4);
          second = warp_sum((s0 + s1) + (s3 + s4));
        }
      }
      if (!x.whole || (!greedy && !(second < INFINITY))) {
        if (!x.whole) {
#pragma unroll 1
          for (int i = 0; i < kLoads<T>; ++i) {
            float v[kVec<T>];
            r.load(g0 + i * 32, v);
#pragma unroll
            for (int k = 0; k < kVec<T>; ++k) top = fmaxf(top, v[k]);
          }
          top = warp_max(top);
        }
        int at = 0x7fffffff;
        second = 0.f;
#pragma unroll 1
        for (int i = 0; i < kLoads<T> && top > -INFINITY; ++i) {
          float v[kVec<T>];
          r.load(g0 + i * 32, v);
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) {
            if (v[k] == top) at = min(at, (g0 + i * 32) * kVec<T> - r.mis + k);
            second += weight32(v[k], top, c);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
        second = warp_sum(second);
        if (greedy) second = __int_as_float(at);
      }
      if (lane == 0) a.part[((size_t)x.row * 2 + x.which) * a.pieces + x.piece] = make_float2(top, second);
    };
    uint4 raw0[kLoads<T>], raw1[kLoads<T>];
    Unit x0, x1;
    if (left) x0 = fetch(raw0);
    else continue;
    while (true) {
      const bool more = left != 0;
      if (more) x1 = fetch(raw1);
      work(x0, raw0);
      if (!more) break;
      const bool again = left != 0;
      if (again) x0 = fetch(raw0);
      work(x1, raw1);
      if (!again) break;
    }
  }
}

// ------------------------------------------------------------------------------------- decisions
constexpr int kTable = 256;
// log2(e) / T in ways: for e^((x - best) / T) in 64 bits, times kTable as two floats, and as one.
struct Heat {
  double inv;                  // 1 / T
  float hi, lo, c;
  const double* table;         // 2^(i / kTable)
  __device__ __forceinline__ Heat(float heat, const double* table_) : inv(1. / (double)heat), table(table_) {
    c = inverse_heat(heat);
    const double whole = fmin(inv, 1e30) * (kTable * 1.4426950408889634);
    hi = (float)whole, lo = (float)(whole - (double)hi);
  }
};
__device__ __noinline__ double large_weight(float x, float best, double inv) {
  if (x == best) return x == -INFINITY ? 0. : 1.;
  if (x == -INFINITY || best == INFINITY) return 0.;
  return exp(((double)x - (double)best) * inv);
}
// A logit's weight beside the row's largest one, as exactly as it counts (see above).
__device__ __forceinline__ double weight64(float x, float best, const Heat& h) {
  const float d = x - best, e = d * h.c;
  if (!(e < -14.4f) || best == INFINITY) return large_weight(x, best, h.inv);   // (2^-14.4 is e^-10; or e is no number)
  if (e < -120.f) return 0.;                                       // (nothing beside the largest, 2^-100 of all V)
  // d + rest is x - best, n whole and t what is left of (x - best) / T in units of ln 2 / kTable
  const float back = d - x, rest = (x - (d - back)) + (-best - back);
  const float shifted = fmaf(d, h.hi, 12582912.f), n = shifted - 12582912.f;
  const float t = fmaf(rest, h.hi, fmaf(d, h.lo, fmaf(d, h.hi, -n)));
  const float r = t * (0.6931471805599453f / kTable);
  const float p = fmaf(r * r, fmaf(r, 1.f / 6.f, 0.5f), r);        // e^r - 1; r^4 / 24 is below 2e-13
  const int whole = __float_as_int(shifted) - 0x4b400000;          // n
  const double f = h.table[whole & (kTable - 1)];
  const double w = fma(f, (double)p, f);
  return __hiloint2double(__double2hiint(w) + ((whole >> 8) << 20), __double2loint(w));
}
static_assert(kTable == 256, "the shift above");
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

// Loads of a row that are under way together: a lane's groups g, g + 32, ...
template <typename T> struct Ahead {
  uint4 raw[kAhead];
  __device__ __forceinline__ void load(const Row<T>& x, int g, int end) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (g + 32 * i < end && x.whole(g + 32 * i)) raw[i] = x.raw(g + 32 * i);
  }
  __device__ __forceinline__ void get(const Row<T>& x, int i, int g, float (&v)[kVec<T>]) const {      // i: a constant
    if (x.whole(g)) {
      unpack<T>(raw[i], v);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) v[k] = fmaxf(v[k], -INFINITY);
    } else {
      x.load(g, v);
    }
  }
  __device__ __forceinline__ double sum(const Row<T>& x, int g, int end, float best, const Heat& h) const {
    double s = 0.;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (g + 32 * i >= end) break;
      float z[kVec<T>];
      get(x, i, g + 32 * i, z);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) s += weight64(z[k], best, h);
    }
    return s;
  }
};

template <typename T>
__global__ void __launch_bounds__(kDecide, 1) verify_decide_kernel(const VerifyArgs a) {
  __shared__ Total totals[kBatch][2];                 // of the batch's rows: the target's, the draft's
  __shared__ int places[kBatch];                      // greedy: the arg-max
  __shared__ double sums[kWarps][2];
  __shared__ __align__(16) double slots[2][2];
  __shared__ int verdict[2];
  __shared__ double table[kTable];
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
  if (threadIdx.x < kTable) table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
  const Heat h(heat, table);
  // this block's share of a row's groups of 16 bytes, and the warp's of that, in order
  auto block_share = [&](int groups, int& g0, int& g1) {
    const int each = (groups + (int)cl.size - 1) / (int)cl.size;
    g0 = min(groups, (int)cl.rank * each), g1 = min(groups, g0 + each);
  };
  auto share_of = [&](int groups, int& w0, int& w1) {
    int g0, g1;
    block_share(groups, g0, g1);
    const int per = (g1 - g0 + kWarps - 1) / kWarps;
    w0 = min(g1, g0 + warp * per), w1 = min(g1, w0 + per);
  };
  // both rows' sums of weights in 64 bits
  auto exact_totals = [&](int row, bool with_draft, float best, float draft_best, double& P, double& Q) {
    double s[2] = {0., 0.};
    const Row<T> x(a.logits, a.stride, row, a.V), y(with_draft ? a.draft : a.logits, with_draft ? a.draft_stride : a.stride, row, a.V);
    int x0, x1, y0, y1;
    share_of(x.groups(), x0, x1);
    share_of(y.groups(), y0, y1);
    if (!with_draft) y1 = y0;
    Ahead<T> vx, vy;
    for (int gx = x0 + lane, gy = y0 + lane; gx < x1 || gy < y1; gx += 32 * kAhead, gy += 32 * kAhead) {
      vx.load(x, gx, x1);
      vy.load(y, gy, y1);
      s[0] += vx.sum(x, gx, x1, best, h);
      s[1] += vy.sum(y, gy, y1, draft_best, h);
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
        if (!which) places[i] = best == -INFINITY ? 0 : min(max(at, 0), a.V - 1);
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
  if (with_draft && !exact) exact_totals(row, true, best, draft_best, P, Q);
  const Row<T> x(a.logits, a.stride, row, a.V), y(with_draft ? a.draft : a.logits, with_draft ? a.draft_stride : a.stride, row, a.V);
  const int d = refused ? fresh_index(a.tokens + row + 1) : -1;
  // (where nothing is taken off p its sum need not be known)
  const double inv_p = !with_draft ? 1. : P > 0. ? 1. / P : 0., inv_q = Q > 0. ? 1. / Q : 0.;
  int w0, w1;
  share_of(x.groups(), w0, w1);
  // a group's weights: without `whole` what p has more than q
  const bool side_by_side = y.mis == x.mis;
  auto rest = [&](int g, const float (&v)[kVec<T>], const float (&z)[kVec<T>], bool whole, double (&w)[kVec<T>]) {
    const int j = g * kVec<T> - x.mis;
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) {
      w[k] = weight64(v[k], best, h) * inv_p;
      if (with_draft && !whole) w[k] = fmax(w[k] - weight64(z[k], draft_best, h) * inv_q, 0.);
      else if (refused && !whole && j + k == d) w[k] = 0.;
    }
  };
  // what is taken off it: the draft's logits of the same tokens
  auto beside = [&](int g, float (&z)[kVec<T>]) {
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) z[k] = y.at(g * kVec<T> - x.mis + k);
  };
  const double u = fmin(fmax((double)fresh(a.u + rows.end - 1), 0.), 1. - 0x1p-24);     // (whatever is handed in)
  for (int whole = 0; whole < 2; ++whole) {           // (where nothing is left of p - q: p itself)
    double mine = 0.;
    Ahead<T> vx, vy;
    for (int g = w0 + lane; g < w1; g += 32 * kAhead) {
      vx.load(x, g, w1);
      if (with_draft && side_by_side) vy.load(y, g, w1);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (g + 32 * i >= w1) break;
        float v[kVec<T>], z[kVec<T>] = {};
        double w[kVec<T>];
        vx.get(x, i, g + 32 * i, v);
        if (with_draft && side_by_side) vy.get(y, i, g + 32 * i, z);
        else if (with_draft) beside(g + 32 * i, z);
        rest(g + 32 * i, v, z, whole, w);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) mine += w[k];
      }
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
      // its share again, in smaller ones for all of the block's warps
      int b0, b1;
      block_share(x.groups(), b0, b1);
      const int per = (b1 - b0 + kWarps - 1) / kWarps, seg0 = min(b1, b0 + owner * per), seg1 = min(b1, seg0 + per),
                sub = (seg1 - seg0 + kWarps - 1) / kWarps;
      const int s0 = min(seg1, seg0 + warp * sub), s1 = min(seg1, s0 + sub);
      auto weights_at = [&](int g, double (&w)[kVec<T>]) {
        if (g < s1) {
          float v[kVec<T>], z[kVec<T>] = {};
          x.load(g, v);
          if (with_draft && side_by_side) y.load(g, z);
          else if (with_draft) beside(g, z);
          rest(g, v, z, whole, w);
        } else {
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) w[k] = 0.;
        }
      };
      double part = 0.;
      for (int g = s0; g < s1; g += 32) {
        double w[kVec<T>];
        weights_at(g + lane, w);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) part += w[k];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += shfl_xor(part, o);
      if (lane == 0) sums[warp][1] = part;
      __syncthreads();
      int finder = -1;
      double run = 0.;
      ahead = owner_ahead;
      for (int w = 0; w < kWarps; ++w) {
        if (sums[w][1] > 0. && (finder < 0 || ahead < target)) finder = w, run = ahead;
        ahead += sums[w][1];
      }
      if (warp == finder) {
        int last = -1;
        bool found = false;
        for (int g = s0; g < s1 && !found; g += 32) {
          double w[kVec<T>], mine_here = 0.;
          weights_at(g + lane, w);
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) mine_here += w[k];
          double upto = mine_here;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += up;
          }
          double at = run + (upto - mine_here);
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
// vocabulary, requests, scratch and its bytes, SMs, stream.
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
  const int sms = (int)w[i++];
  cudaStream_t stream = (cudaStream_t)ptr();
  if (a.B <= 0) return 0;
  const bool half = type == GF_BF16;
  a.pieces = (a.V + (half ? kVec<bf16> : kVec<float>) - 1 + kPiece - 1) / kPiece;
  if ((long long)a.R * 2 * a.pieces * 8 > room) return -5;
  int rc = 0;
  if (a.R > 0) {
    const long long units = (long long)a.R * a.pieces * (a.draft ? 2 : 1), most = (long long)sms * kScanBlocks;
    const long long blocks = (units + kScan / 32 - 1) / (kScan / 32);
    rc = launch_kernel(half ? verify_scan_kernel<bf16> : verify_scan_kernel<float>, dim3((unsigned)(blocks < most ? blocks : most)),
                       dim3(kScan), 0, stream, a);
  }
  if (rc) return rc;
  static OncePerDevice attrs;
  rc = attrs.run([&] {
    const cudaError_t e = cudaFuncSetAttribute(verify_decide_kernel<bf16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e != cudaSuccess ? e
                            : cudaFuncSetAttribute(verify_decide_kernel<float>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (rc) return rc;
  const char* env = getenv("GF_CLUSTER");
  const int cluster = env ? atoi(env) : a.B <= 4 ? 16 : a.B <= 18 ? 8 : 4;
  return launch_kernel_cluster_dims(half ? verify_decide_kernel<bf16> : verify_decide_kernel<float>, dim3(a.B * cluster),
                                    dim3(kDecide), 0, stream, cluster, true, a);
}
