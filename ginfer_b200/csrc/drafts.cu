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
//    from the one row that it needs: from the pieces' sums and the piece that the token is in, or, where q is taken off p, from
//    both rows, read again.
// Sums and weights in 32 bits are enough nearly always: the numbers that are returned are whole, and a comparison says so itself when
// its two sides are within what 32 bits may be off (kMargin, kDrawMargin).  Then, and then alone, the rows' sums are
// taken again with weights in 64 bits.
#include "common.cuh"
#include "tc_common.cuh"

namespace gf {
namespace {

constexpr int kLoads = 8;                               // 16-byte loads a lane of a piece
constexpr int kPiece = 1024;                            // the least logits of a piece
constexpr int kScan = 256, kScanBlocks = 2;             // threads of a scanning block, blocks an SM
constexpr int kSearch = 1024;                           // requests whose first rows a scanning block keeps
constexpr int kDecide = 256, kWarps = kDecide / 32, kBatch = 32;      // rows whose sums are at hand at a time
// Blocks of a request: 8 up to a number of requests, else 4 (2, 5, 6 and 16 are slower): the more logits a draw goes through, a
// row of the target and one of the drafter, the longer twice the blocks are worth their starts and barriers.  8 / 4, us, requests of
// 4 drafts: 152,064 logits and a drafter, 64 requests 134 / 155, 128 220 / 230, 160 257 / 257, 256 399 / 378, the same in bfloat16
// 124 / 135, 195 / 193 (128), 353 / 311 (256); of 1 draft 77 / 115, 115 / 134, 220 / 213, of 8 185 / 210, 320 / 324, 599 / 558; 100,000 logits, 64
// 102 / 108, 128 166 / 162; 64,000, 64 68 / 75, 96 92 / 92, 128 122 / 112; 32,003, 32 36 / 42, 64 48 / 45, 128 80 / 68; 8,000, 32 22 / 21, 64
// 31 / 24; look-ups, 152,064, 32 50 / 63, 64 80 / 79, 128 136 / 118; 32,003, 32 26 / 27, 64 40 / 33.
__host__ inline int blocks_of_request(int requests, int vocabulary, bool drafter) {
  return requests > 28 + vocabulary / (drafter ? 1500 : 3000) ? 4 : 8;
}
constexpr int kAhead = 4;                               // loads of a row that are under way
// Relative error that numbers in 32 bits may have.  A weight's: 3.5 roundings of its exponent (difference, 1 / T, product), 1.45e-7
// of it in the weight, and 2^-22 of each exponential; what is summed weighs its own exponents, log2 V = 28 at most in the mean,
// 4e-6.  A piece's sum: 64 roundings at most, 3.8e-6; pieces are added up in 64 bits.  So a row's sum is off by 9e-6, a draft's
// weight, compared down to 1e-30, an exponent of 100, by 1.5e-5, and u q(d) beside p(d) by 5e-5.
constexpr double kMargin = 8e-5;
// The same of a running sum beside u times the whole, in parts of 1: 5e-6 for its weights and 9e-6 for the row's sum, of p and of q: 2.8e-5.
constexpr double kDrawMargin = 4e-5;
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
template <typename T> constexpr int kPieceOf = 32 * kLoads * kVec<T>;              // logits of a piece
static_assert(kPieceOf<float> == kPiece, "the least");
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
  // The same for what is read in passing, past L1, too: it leaves L2 first.  (`once`: a policy that says so.)
  __device__ __forceinline__ uint4 passing(int g, uint64_t once) const {
    uint4 v;
    asm volatile("ld.global.cg.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(x + (g * kVec<T> - mis)), "l"(once));
    return v;
  }
  // A group that the row begins or ends in, or one outside it: -inf in places outside.
  __device__ __forceinline__ uint4 pieced(int g) const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(at(g * kVec<T> - mis + i));
      } else {
        const int j = g * kVec<T> - mis + 2 * i;
        w[i] = (__float_as_uint(at(j)) >> 16) | (__float_as_uint(at(j + 1)) & 0xffff0000u);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
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
// A piece with care, by a warp: one with a weight that is no number.  (Out of line: the others keep their registers.)
template <typename T>
__device__ __noinline__ float careful_sum(const Row<T>& r, int g0, float top, float c) {
  float sum = 0.f;
#pragma unroll 2
  for (int i = 0; i < kLoads; ++i) {
    float v[kVec<T>];
    r.load(g0 + i * 32, v);
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) sum += weight32(v[k], top, c);
  }
  return warp_sum(sum);
}
// The largest of a group's logits (a NaN never is).
template <typename T> __device__ __forceinline__ float group_max(const uint4& raw) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
}

// A warp takes a piece after the other, the loads of the next one under way while it works on one.  Memory bounds it: 512 rows of
// 152,064 logits in 32 bits, 311 MB, 55 us, 5.65 TB/s; 1,011 MB in bfloat16 191 us, 5.3 TB/s (twice the exponentials a byte).
template <typename T>
__global__ void __launch_bounds__(kScan, kScanBlocks) verify_scan_kernel(const VerifyArgs a) {
  __shared__ int starts[kSearch + 1];
  constexpr int GROUPS = 32 * kLoads;
  const int lane = threadIdx.x & 31;
  uint64_t once;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
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
      // (turned by the row: a row's last piece, which costs more, is not always the same warps')
      my_piece = (int)((at - (long long)my_row * a.pieces + my_row) % a.pieces);
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
    };
    auto fetch = [&](uint4 (&raw)[kLoads]) {            // the next of the ballot's
      const int who = __ffs(left) - 1;
      left &= left - 1;
      Unit x{__shfl_sync(0xffffffffu, my_row, who), __shfl_sync(0xffffffffu, my_which, who),
             __shfl_sync(0xffffffffu, my_piece, who), __shfl_sync(0xffffffffu, my_heat, who)};
      const Row<T> r(x.which ? a.draft : a.logits, x.which ? a.draft_stride : a.stride, x.row, a.V);
      const int g0 = x.piece * GROUPS + lane;
      if (r.whole(x.piece * GROUPS) && r.whole(x.piece * GROUPS + GROUPS - 1)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) raw[i] = r.passing(g0 + i * 32, once);
      } else {
        const uint32_t none = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) raw[i] = r.whole(g0 + i * 32) ? r.passing(g0 + i * 32, once) : make_uint4(none, none, none, none);
        // (the row's first and last group)
        const int first = r.mis ? 0 : -1, last = (a.V + r.mis) % kVec<T> ? r.groups() - 1 : -1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          if (g0 + i * 32 == first || g0 + i * 32 == last) raw[i] = r.pieced(g0 + i * 32);
      }
      return x;
    };
    auto work = [&](const Unit& x, const uint4 (&raw)[kLoads]) {
      const Row<T> r(x.which ? a.draft : a.logits, x.which ? a.draft_stride : a.stride, x.row, a.V);
      const bool greedy = !(x.heat > 0.f);
      const float c = inverse_heat(x.heat);
      const int g0 = x.piece * GROUPS + lane;
      float top = -INFINITY, second = 0.f;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) top = fmaxf(top, group_max<T>(raw[i]));
      top = warp_max(top);
      if (greedy) {
        int at = 0x7fffffff;
#pragma unroll
        for (int i = kLoads - 1; i >= 0; --i) {
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
        for (int i = 0; i < kLoads; ++i) {
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
      if (!greedy && !(second < INFINITY)) second = top > -INFINITY ? careful_sum<T>(r, g0, top, c) : 0.f;
      if (lane == 0) a.part[((size_t)x.row * 2 + x.which) * a.pieces + x.piece] = make_float2(top, second);
    };
    uint4 raw0[kLoads], raw1[kLoads];
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
__device__ __forceinline__ double shfl_xor(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += shfl_xor(v, o);
  return v;
}

// Weights in 64 bits: 2^y for y = (x - best) log2(e) / T as 2^(n / kTable), n the nearest whole number to kTable y, from a
// table, times the power series of 2^f, |f| <= 1 / (2 kTable), to the sixth power (what is cut off is at most 4.4e-16 of it).
// The table has as many entries as there are pairs of banks: a warp's look-ups never wait for one another.  INFINITE: for rows
// whose largest logit is infinite; the others do without its comparisons.  (64 entries, the fifth power and the comparisons
// everywhere: 139 us for 64 requests of 152,064 logits, 132 like this.)
constexpr int kTable = 16;
template <bool INFINITE> struct Exact {
  double c;                    // log2(e) / T
  float c32;
  const double* table;         // 2^(i / kTable)
  __device__ __forceinline__ Exact(float heat, const double* table_)
      : c(fmin(1.4426950408889634 / (double)heat, 1e30)), c32((float)c), table(table_) {}
  // A logit's weight beside the row's largest one; below 2^-120, and for a NaN, nothing.  (Without branches, so that several
  // are under way.)
  __device__ __forceinline__ double operator()(float x, float best) const {
    constexpr double kShift = 6755399441055744.0 / kTable;           // 1.5 * 2^52 / kTable: n in the last bits
    const double d = (double)x - (double)best, at = fma(d, c, kShift), f = fma(d, c, -(at - kShift));
    double p = fma(f, 0.00015403530393381608, 0.0013333558146428443);                  // ln(2)^k / k!
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    const int n = __double2loint(at);
    const double y = p * table[n & (kTable - 1)];
    const double z = __hiloint2double(__double2hiint(y) + ((n >> 4) << 20), __double2loint(y));
    // (the product is no number for a NaN and for -inf at a temperature of infinity)
    const double w = (x - best) * c32 >= -120.f ? z : 0.;
    if constexpr (INFINITE) return x == best ? (x > -INFINITY ? 1. : 0.) : w;
    return w;
  }
};
static_assert(kTable == 16, "the shift above");

// What a row's weights are relative to, and their sum.
struct Total {
  float best, sum;
};
// All threads of a cluster's blocks.  (The barrier's instructions want a warp as one; what stands in front of them are stores of
// single lanes.)
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  cluster_sync();
}
struct Cluster {
  uint32_t rank, size;
  int round;
  double (*slots)[2];          // [2][2] of this block
  // Both numbers' sums over the cluster's blocks, in the order of their ranks; `before`: what the blocks ahead of this one have of the
  // first.  By all threads; `mine` is the block's, known to thread 0.
  __device__ __forceinline__ void add(double mine0, double mine1, double& all0, double& all1, double& before) {
    double* at = slots[round & 1];
    if (threadIdx.x == 0) at[0] = mine0, at[1] = mine1;
    cluster_meet();
    // (a lane a block)
    double x = 0., y = 0.;
    const uint32_t lane = threadIdx.x & 31;
    if (lane < size) {
      const uint32_t from = dsmem_addr(smem_u32(at), lane);
      asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(x), "=d"(y) : "r"(from) : "memory");
    }
    all0 = all1 = before = 0.;
    for (uint32_t r = 0; r < size; ++r) {
      if (r == rank) before = all0;
      all0 += __shfl_sync(0xffffffffu, x, r), all1 += __shfl_sync(0xffffffffu, y, r);
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
};

// What a block needs for one request's row.
template <typename T> struct Draw {
  const VerifyArgs& a;
  Cluster& cl;
  double (*sums)[2];           // [kWarps][2]
  Row<T> x, y;                 // the target's row and the draft's (the target's again where there is none)
  bool with_draft, side_by_side;
  float best, draft_best;
  int d;                       // the token that is taken out; -1: none
  int b0, b1, per, w0, w1;     // this block's groups, a warp's share of them, this warp's
  __device__ __forceinline__ Draw(const VerifyArgs& a_, Cluster& cl_, double (*sums_)[2], int row, bool draft_, float best_,
                                  float draft_best_, int d_)
      : a(a_), cl(cl_), sums(sums_), x(a_.logits, a_.stride, row, a_.V),
        y(draft_ ? a_.draft : a_.logits, draft_ ? a_.draft_stride : a_.stride, row, a_.V), with_draft(draft_),
        best(best_), draft_best(draft_best_), d(d_) {
    side_by_side = y.mis == x.mis;
    const int groups = x.groups(), each = (groups + (int)cl.size - 1) / (int)cl.size, warp = threadIdx.x >> 5;
    b0 = min(groups, (int)cl.rank * each), b1 = min(groups, b0 + each);
    per = (b1 - b0 + kWarps - 1) / kWarps;
    w0 = min(b1, b0 + warp * per), w1 = min(b1, w0 + per);
  }
  // Four of a group's logits: in 32 bits all of them.
  static __device__ __forceinline__ void quarter(const uint4& raw, int h, float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
      unpack<T>(raw, v);
    } else {
      const uint32_t w0 = h ? raw.z : raw.x, w1 = h ? raw.w : raw.y;
      v[0] = __uint_as_float(w0 << 16), v[1] = __uint_as_float(w0 & 0xffff0000u);
      v[2] = __uint_as_float(w1 << 16), v[3] = __uint_as_float(w1 & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void beside(int g, float (&z)[kVec<T>]) const {
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) z[k] = y.at(g * kVec<T> - x.mis + k);
  }
  // Calls f(a logit's number, logits from there, the draft's logits) for the groups g, g + 32, ... up to `end`.  LONG: f is long (64
  // bits) and knows what a NaN is: its code stands here once, for four logits at a time, with the next group's loads under way;
  // else kAhead groups' are.
  template <bool LONG, typename F> __device__ __forceinline__ void each_group(int g, int end, F&& f) const {
    if constexpr (LONG) {
      uint4 rx{}, ry{};
      const bool both = with_draft && side_by_side;
      auto fetch = [&](int h) {
        if (h < end && x.whole(h)) {
          rx = x.raw(h);
          if (both) ry = y.raw(h);
        }
      };
      fetch(g);
#pragma unroll 1
      for (; g < end; g += 32) {
        if (!x.whole(g)) {
          rx = x.pieced(g);
          if (both) ry = y.pieced(g);
        }
        const uint4 vx = rx, vy = ry;
        fetch(g + 32);
#pragma unroll 1
        for (int h = 0; h < kVec<T> / 4; ++h) {
          const int j = g * kVec<T> - x.mis + 4 * h;
          float v[4], z[4] = {};
          quarter(vx, h, v);
          if (both) quarter(vy, h, z);
          else if (with_draft)
#pragma unroll
            for (int k = 0; k < 4; ++k) z[k] = y.at(j + k);
          f(j, v, z);
        }
      }
    } else {
      Ahead<T> vx, vy;
      for (; g < end; g += 32 * kAhead) {
        vx.load(x, g, end);
        if (with_draft && side_by_side) vy.load(y, g, end);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (g + 32 * i >= end) break;
          float v[kVec<T>], z[kVec<T>] = {};
          vx.get(x, i, g + 32 * i, v);
          if (with_draft && side_by_side) vy.get(y, i, g + 32 * i, z);
          else if (with_draft) beside(g + 32 * i, z);
          f((g + 32 * i) * kVec<T> - x.mis, v, z);
        }
      }
    }
  }
  // The block's total of what the threads have, in the order of the warps; `sums` keeps theirs.
  __device__ __forceinline__ double block_total(double mine, int which) const {
    mine = warp_total(mine);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5][which] = mine;
    __syncthreads();
    double t = 0.;
    for (int w = 0; w < kWarps; ++w) t += sums[w][which];
    return t;
  }
  // Both rows' sums of weights in 64 bits.
  template <bool INFINITE> __device__ __forceinline__ void totals(const Exact<INFINITE>& e, double& P, double& Q) const {
    double s0 = 0., s1 = 0., unused;
    each_group<true>(w0 + (threadIdx.x & 31), w1, [&](int, const float (&v)[4], const float (&z)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s0 += e(v[k], best);
        if (with_draft) s1 += e(z[k], draft_best);
      }
    });
    const double m0 = block_total(s0, 0), m1 = block_total(s1, 1);
    cl.add(m0, m1, P, Q, unused);
  }
  // The first index at which the running sum of `weight(v, z, j)` reaches u times the whole, in the block that has it (-1 elsewhere, and
  // everywhere where there is no weight); `low` and `high`: the sum in front of it and with it, as parts of the whole.  By the
  // whole cluster.
  template <bool LONG, typename W>
  __device__ __forceinline__ int search(double u, const W& weight, double& total, double& target, double& low, double& high) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double mine = 0., before, unused;
    each_group<LONG>(w0 + lane, w1, [&](int j, const auto& v, const auto& z) {
      auto s = weight(v[0], z[0], j);
#pragma unroll
      for (int k = 1; k < (int)(sizeof(v) / sizeof(float)); ++k) s += weight(v[k], z[k], j + k);
      mine += (double)s;
    });
    const double block = block_total(mine, 0);
    cl.add(block, 0., total, unused, before);
    target = u * total;
    // the block, in it the warp's share, and in that a smaller share, in which the sum is reached (the last one that weighs
    // anything, should rounding leave it short)
    if (!(total > 0.) || !(block > 0.) || !(before < target || before == 0.) || !(before + block >= target || before + block == total))
      return -1;
    auto pick = [&](int which, double& ahead) {
      int owner = -1;
      double at = ahead;
      for (int w = 0; w < kWarps; ++w) {
        const double s = sums[w][which];
        if (s > 0. && (owner < 0 || at < target)) owner = w, ahead = at;
        at += s;
      }
      return owner;
    };
    const int owner = pick(0, before);
    const int seg0 = min(b1, b0 + owner * per), seg1 = min(b1, seg0 + per), sub = (seg1 - seg0 + kWarps - 1) / kWarps;
    const int s0 = min(seg1, seg0 + warp * sub), s1 = min(seg1, s0 + sub);
    double part = 0.;
    each_group<true>(s0 + lane, s1, [&](int j, const float (&v)[4], const float (&z)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        part += (double)(LONG ? weight(v[k], z[k], j + k) : weight(fmaxf(v[k], -INFINITY), fmaxf(z[k], -INFINITY), j + k));
    });
    block_total(part, 1);
    const int finder = pick(1, before);
    if (warp != finder) return -1;
    double run = before;
    int last = -1;
    for (int g = s0; g < s1; g += 32) {
      float v[kVec<T>], z[kVec<T>] = {};
      double w[kVec<T>], here = 0.;
      if (g + lane < s1) {
        x.load(g + lane, v);
        if (with_draft && side_by_side) y.load(g + lane, z);
        else if (with_draft) beside(g + lane, z);
      }
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) {
        w[k] = g + lane < s1 ? (double)weight(v[k], z[k], (g + lane) * kVec<T> - x.mis + k) : 0.;
        here += w[k];
      }
      double upto = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      double at = run + (upto - here), lo = 0., hi = 0.;
      int hit = -1, latest = -1;
      double latest_lo = 0., latest_hi = 0.;
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) {
        const double from = at;
        at += w[k];
        if (w[k] > 0.) {
          latest = (g + lane) * kVec<T> - x.mis + k, latest_lo = from, latest_hi = at;
          if (hit < 0 && at >= target) hit = latest, lo = from, hi = at;
        }
      }
      const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, latest >= 0);
      if (hits) {
        const int who = __ffs(hits) - 1;
        low = __shfl_sync(0xffffffffu, lo, who), high = __shfl_sync(0xffffffffu, hi, who);
        return __shfl_sync(0xffffffffu, hit, who);
      }
      if (some) {
        const int who = 31 - __clz(some);
        low = __shfl_sync(0xffffffffu, latest_lo, who), high = __shfl_sync(0xffffffffu, latest_hi, who);
        last = __shfl_sync(0xffffffffu, latest, who);
      }
      run += __shfl_sync(0xffffffffu, upto, 31);
    }
    return last;
  }
};

// In 64 bits, by the whole cluster.  (Out of line: what nearly every request needs keeps its registers.)
// Whether u q(d) < p(d).
template <typename T, bool INFINITE>
__device__ __noinline__ bool exactly_stays(const VerifyArgs& a, Cluster& cl, double (*sums)[2], const double* tables, float heat,
                                           int row, float best, float draft_best) {
  const Draw<T> r(a, cl, sums, row, a.draft != nullptr, best, draft_best, -1);
  const Exact<INFINITE> e(heat, tables);
  const int d = fresh_index(a.tokens + row + 1);
  double P, Q;
  r.totals(e, P, Q);
  const double p = e(r.x.at(d), r.best) / P, q = a.draft ? (Q > 0. ? e(r.y.at(d), r.draft_best) / Q : 0.) : 1.;
  return (double)fresh(a.u + row) * q < p;
}
// The token behind the drafts that stay, in the block that has it; -1 elsewhere.  `none`: the row has no weight at all.
template <typename T, bool INFINITE>
__device__ __noinline__ int exactly_drawn(const VerifyArgs& a, Cluster& cl, double (*sums)[2], const double* tables, float heat,
                                          int row, bool with_draft, float best, float draft_best, int d, double u, bool& none) {
  const Draw<T> r(a, cl, sums, row, with_draft, best, draft_best, d);
  const Exact<INFINITE> e(heat, tables);
  double P = 1., Q = 1., total = 0., target, low, high;
  if (with_draft) r.totals(e, P, Q);
  const double inv_p = P > 0. ? 1. / P : 0., inv_q = Q > 0. ? 1. / Q : 0.;
  none = false;
  for (int whole = 0; whole < 2; ++whole) {           // (where nothing is left of p - q: p itself)
    auto weight = [&](float v, float z, int j) {
      double w = e(v, r.best) * inv_p;
      if (with_draft && !whole) w = fmax(w - e(z, r.draft_best) * inv_q, 0.);
      return j == r.d && !whole ? 0. : w;
    };
    const int token = r.template search<true>(u, weight, total, target, low, high);
    if (total > 0.) return token;
  }
  none = true;
  return -1;
}

// Latency bounds it: a request's rows, its pieces' totals and its verdict take 4.6 us, a draw in 32 bits 8 more, one in 64 bits 30 to
// 45 (64 requests of 152,064 logits: 78 us with 15 of them in 64 bits, 30 with none).  In 64 bits a request with a draft model takes
// 38,000 weights a block and pass, which two warps a scheduler work on: instructions that are not there yet and waits for results
// keep them at a third of its rate.  Blocks of 512 threads 149 us for the call, of 256 132; four a SM 139 (registers), two or three 132.
template <typename T>
__global__ void __launch_bounds__(kDecide, 2) verify_decide_kernel(const VerifyArgs a) {
  __shared__ Total totals[kBatch][2];                 // of the batch's rows: the target's, the draft's
  __shared__ float drafted[kBatch][2];                // the logits that both give the draft
  __shared__ int places[kBatch];                      // greedy: the arg-max
  __shared__ double sums[kWarps][2];
  __shared__ __align__(16) double slots[2][2];
  __shared__ int verdict[2];
  __shared__ double tables[kTable];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Cluster cl{cluster_rank(), 0, 0, slots};
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cl.size));
  const int b = blockIdx.x / cl.size;
  pdl_trigger();
  pdl_wait();
  const Span rows = rows_of(a, b);
  const int n = rows.end - rows.first;
  const float heat = fresh(a.temperature + b);
  if (n == 0) {                                       // (the whole cluster)
    if (cl.rank == 0 && threadIdx.x == 0) a.accepted[b] = 0, a.next[b] = -1;
    return;
  }
  const bool greedy = !(heat > 0.f);
  const float c = inverse_heat(heat);
  bool have_tables = false;
  auto make_tables = [&] {
    if (!have_tables)
      for (int i = threadIdx.x; i < kTable; i += kDecide) tables[i] = exp2((double)i / kTable);
    __syncthreads();
    have_tables = true;
  };

  int stop = n - 1, in_batch = 0;
  bool refused = false;
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    // the batch's totals, a warp a row
    const int here = min(kBatch, n - i0);
    __syncthreads();
    for (int k = warp; k < 2 * here; k += kWarps) {
      const int i = k >> 1, which = k & 1, row = rows.first + i0 + i;
      if (which && (!a.draft || greedy || i0 + i == n - 1)) continue;
      const float2* part = a.part + ((size_t)row * 2 + which) * a.pieces;
      // (-inf for a draft that is none)
      float own = -INFINITY;
      if (i0 + i < n - 1)
        own = Row<T>(which ? a.draft : a.logits, which ? a.draft_stride : a.stride, row, a.V).at(fresh_index(a.tokens + row + 1));
      float best = -INFINITY;
      double sum = 0.;                                // (there may be 2^18 pieces)
      int at = 0x7fffffff;
      for (int q0 = lane; q0 < a.pieces; q0 += 32 * 8) {
        float2 y[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) y[q] = q0 + 32 * q < a.pieces ? __ldcg(part + q0 + 32 * q) : make_float2(-INFINITY, 0.f);
        float top = best;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (greedy && q0 + 32 * q < a.pieces && (y[q].x > top || (y[q].x == top && __float_as_int(y[q].y) < at)))
            at = __float_as_int(y[q].y);
          top = fmaxf(top, y[q].x);
        }
        if (!greedy && top > -INFINITY) {
          sum = best > -INFINITY ? sum * (double)weight32(best, top, c) : 0.;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (y[q].x > -INFINITY) sum += (double)(y[q].y * weight32(y[q].x, top, c));
        }
        best = top;
      }
      if (greedy) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float ob = __shfl_xor_sync(0xffffffffu, best, o);
          const int oa = __shfl_xor_sync(0xffffffffu, at, o);
          if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
        }
      } else {
        const float top = warp_max(best);
        sum = warp_total(best > -INFINITY ? sum * (double)weight32(best, top, c) : 0.);
        best = top;
      }
      if (lane == 0) {
        totals[i][which] = {best, (float)sum}, drafted[i][which] = own;
        if (!which) places[i] = best == -INFINITY ? 0 : min(max(at, 0), a.V - 1);
      }
    }
    __syncthreads();
    // the first row of the batch at which it ends: 0 the draft stays, 1 it does not, 2 too near to say, 3 the last row
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
            const float xd = drafted[i][0];
            if (greedy) {
              what = fresh_index(a.tokens + row + 1) == places[i] ? 0 : 1;
            } else if (!(xd > -INFINITY) || !(totals[i][0].sum > 0.f)) {
              what = 1;
            } else {
              const float p = weight32(xd, totals[i][0].best, c) / totals[i][0].sum;
              float q = 1.f;
              if (a.draft) {
                const float yd = drafted[i][1];
                q = totals[i][1].sum > 0.f && yd > -INFINITY ? weight32(yd, totals[i][1].best, c) / totals[i][1].sum : 0.f;
              }
              const float left = fresh(a.u + row) * q;
              what = left < p ? 0 : 1;
              // (numbers that 32 bits do not hold well are not compared, either)
              if (!(fabsf(left - p) > (float)kMargin * fmaxf(left, p) && fmaxf(left, p) > 1e-30f)) what = 2;
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
      if (what == 2) {
        make_tables();
        const Total* t = totals[who];
        const bool infinite = t[0].best == INFINITY || (a.draft && t[1].best == INFINITY);
        if (infinite ? exactly_stays<T, true>(a, cl, sums, tables, heat, rows.first + stop, t[0].best, t[1].best)
                     : exactly_stays<T, false>(a, cl, sums, tables, heat, rows.first + stop, t[0].best, t[1].best)) {
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
  const Total tp = totals[in_batch][0], tq = with_draft ? totals[in_batch][1] : Total{0.f, 0.f};
  const Draw<T> r(a, cl, sums, row, with_draft, tp.best, tq.best, refused && !with_draft ? fresh_index(a.tokens + row + 1) : -1);
  const double u = fmin(fmax((double)fresh(a.u + rows.end - 1), 0.), 1. - 0x1p-24);     // (whatever is handed in)
  double total = 0., target, low = 0., high = 0.;
  if (!with_draft) {
    // from the pieces' sums, every block for itself (one warp): the piece in which the sum is reached, then the token in it
    if (warp == 0) {
      const float2* part = a.part + (size_t)row * 2 * a.pieces;
      const float xd = r.d >= 0 ? drafted[in_batch][0] : -INFINITY;
      const bool out = xd > -INFINITY;
      const float wd = out ? weight32(xd, r.best, c) : 0.f;
      const int d_piece = out ? (r.d + r.x.mis) / kPieceOf<T> : -1;
      total = (double)tp.sum - (double)wd;
      target = u * total;
      int piece = -1;
      double ahead = 0.;
      for (int q0 = 0; q0 < a.pieces && piece < 0; q0 += 32 * 8) {          // (eight neighbours a lane)
        float2 y[8];
        double s[8], mine = 0.;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          y[q] = q0 + 8 * lane + q < a.pieces ? __ldcg(part + q0 + 8 * lane + q) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          s[q] = y[q].x > -INFINITY ? (double)y[q].y * (double)weight32(y[q].x, r.best, c) : 0.;
          if (q0 + 8 * lane + q == d_piece) s[q] = fmax(s[q] - (double)wd, 0.);
          mine += s[q];
        }
        double upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        double at = ahead + (upto - mine), before = at;
        int hit = -1;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (hit < 0) {
            if (s[q] > 0. && at + s[q] >= target) hit = q0 + 8 * lane + q, before = at;
            at += s[q];
          }
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0);
        if (hits) {
          piece = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
          ahead = __shfl_sync(0xffffffffu, before, __ffs(hits) - 1);
        } else {
          ahead += __shfl_sync(0xffffffffu, upto, 31);
        }
      }
      int token = -1;
      if (piece >= 0) {
        constexpr int G = kLoads;
        const int g0 = piece * (kPieceOf<T> / kVec<T>) + lane * G;               // (neighbouring groups a lane: in order)
        uint4 raw[G];
#pragma unroll
        for (int i = 0; i < G; ++i)
          if (r.x.whole(g0 + i)) raw[i] = r.x.raw(g0 + i);
        // (weights are computed twice rather than kept)
        auto weights = [&](int i, float (&w)[kVec<T>]) {
          if (r.x.whole(g0 + i)) unpack<T>(raw[i], w);
          else r.x.load(g0 + i, w);
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) {
            const float v = fmaxf(w[k], -INFINITY);
            w[k] = v > -INFINITY && (g0 + i) * kVec<T> - r.x.mis + k != r.d ? fast_exp2((v - r.best) * c) : 0.f;   // (c: see `sure`)
          }
        };
        double sums_of[G], here = 0.;
#pragma unroll
        for (int i = 0; i < G; ++i) {
          float w[kVec<T>], s = 0.f;
          weights(i, w);
#pragma unroll
          for (int k = 0; k < kVec<T>; ++k) s += w[k];
          sums_of[i] = s, here += sums_of[i];
        }
        double upto = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        double at = ahead + (upto - here), lo = 0., hi = 0.;
        int hit = -1;
#pragma unroll
        for (int i = 0; i < G; ++i) {
          if (hit < 0 && sums_of[i] > 0. && at + sums_of[i] >= target) {
            float w[kVec<T>];
            weights(i, w);
            double run = at;
#pragma unroll
            for (int k = 0; k < kVec<T>; ++k) {
              if (w[k] > 0.f && hit < 0) {
                lo = run, hi = run + (double)w[k];
                if (hi >= target) hit = (g0 + i) * kVec<T> - r.x.mis + k;
              }
              run += (double)w[k];
            }
          }
          at += sums_of[i];
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0);
        if (hits) {
          const int who = __ffs(hits) - 1;
          token = __shfl_sync(0xffffffffu, hit, who);
          low = __shfl_sync(0xffffffffu, lo, who), high = __shfl_sync(0xffffffffu, hi, who);
        }
      }
      // (off by a part of all of p, which `total` is where no draft is taken out)
      const double room = kDrawMargin * (double)tp.sum;
      // (Nothing in front of the token: whatever the target is, it is reached there.  Behind the piece that the draft is taken out of
      // that cannot be said: what is beside the draft there may be lost in its sum.)
      const bool first = low == 0. && target > 0. && (d_piece < 0 || piece <= d_piece);
      const bool sure = token >= 0 && tp.best < INFINITY && c > 0.f && (target - low > room || first) && high - target > room;
      if (lane == 0) verdict[0] = sure ? token : -1;
    }
    __syncthreads();
    if (verdict[0] >= 0) {
      if (cl.rank == 0 && threadIdx.x == 0) a.accepted[b] = stop, a.next[b] = verdict[0];
      if (cl.round) cluster_meet();
      return;
    }
  } else {
    // from both rows, in 32 bits
    const float inv_p = tp.sum > 0.f ? 1.f / tp.sum : 0.f, inv_q = tq.sum > 0.f ? 1.f / tq.sum : 0.f;
    auto weight = [&](float v, float z, int) {
      const float p = fast_exp2((v - r.best) * c) * inv_p, q = fast_exp2((z - r.draft_best) * c) * inv_q;
      return fmaxf(p - q, 0.f);
    };
    const bool plain = tp.sum > 0.f && tq.sum > 0.f && tp.best < INFINITY && tq.best < INFINITY && c > 0.f;
    int token = -1;
    if (plain) token = r.template search<false>(u, weight, total, target, low, high);
    const bool sure = token >= 0 && target - low > kDrawMargin && high - target > kDrawMargin;
    // whether some block is sure, known to all
    if (threadIdx.x == 0) verdict[0] = 0;
    __syncthreads();
    if (sure && lane == 0) {
      verdict[0] = 1;
      a.accepted[b] = stop, a.next[b] = token;
    }
    __syncthreads();
    double found, unused0, unused1;
    cl.add((double)verdict[0], 0., found, unused0, unused1);
    if (found > 0.) {
      cluster_meet();          // (nobody leaves while another reads its sums)
      return;
    }
  }
  // ---- in 64 bits
  make_tables();
  bool none;
  const bool infinite = tp.best == INFINITY || tq.best == INFINITY;
  const int token = infinite ? exactly_drawn<T, true>(a, cl, sums, tables, heat, row, with_draft, tp.best, tq.best, r.d, u, none)
                             : exactly_drawn<T, false>(a, cl, sums, tables, heat, row, with_draft, tp.best, tq.best, r.d, u, none);
  if (token >= 0 && lane == 0) a.accepted[b] = stop, a.next[b] = token;
  if (none && cl.rank == 0 && threadIdx.x == 0) a.accepted[b] = stop, a.next[b] = 0;      // (a row without a number)
  cluster_meet();              // (nobody leaves while another reads its sums)
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
  const int piece = half ? kPieceOf<bf16> : kPieceOf<float>;
  a.pieces = (a.V + (half ? kVec<bf16> : kVec<float>) - 1 + piece - 1) / piece;
  if ((long long)a.R * 2 * a.pieces * 8 > room) return -5;
  int rc = 0;
  if (a.R > 0) {
    const long long units = (long long)a.R * a.pieces * (a.draft ? 2 : 1), most = (long long)sms * kScanBlocks;
    const long long blocks = (units + kScan / 32 - 1) / (kScan / 32);
    rc = launch_kernel(half ? verify_scan_kernel<bf16> : verify_scan_kernel<float>, dim3((unsigned)(blocks < most ? blocks : most)),
                       dim3(kScan), 0, stream, a);
  }
  if (rc) return rc;
  const int cluster = blocks_of_request(a.B, a.V, a.draft != nullptr);
  return launch_kernel_cluster_dims(half ? verify_decide_kernel<bf16> : verify_decide_kernel<float>, dim3(a.B * cluster),
                                    dim3(kDecide), 0, stream, cluster, true, a);
}
