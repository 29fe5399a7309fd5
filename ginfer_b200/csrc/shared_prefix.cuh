// What the kernels of attention over shared prefixes are told, and how they read it.
//
// Request b has the rows cu[b] .. cu[b + 1] - 1 of q (one row, its own number, without cu); the i-th of n sees the
// prefix of the request's group and the request's own tokens 0 .. length - n + i.  Whatever the tables, lengths and
// starts hold, nothing outside q, the cache and the result is touched: lengths are cut to their tables, rows to q, and
// an entry that is no page of the cache is taken for the nearest.
#pragma once
#include "common.cuh"

namespace gf {

struct PrefixArgs {
  const void* q;
  const void* k;               // pages [pages][page][nkv][hd]
  const void* v;
  const int* prefix_table;     // [G][prefix_stride]
  const int* prefix_lens;      // [G]
  const int* table;            // [B][table_stride]
  const int* lengths;          // [B]
  const int* cu_groups;        // [G + 1], or null: all requests are of group 0
  const int* cu;               // [B + 1], or null: a row a request
  void* out;                   // [T][nh][hd]
  int q_stride, prefix_stride, table_stride, prefix_limit, limit, G, B, T, nh, nkv, hd, page, pages;
  float scale;
};

struct Rows {
  int first, count;
};
__device__ __forceinline__ Rows rows_of(const PrefixArgs& a, int b) {
  if (!a.cu) return {b, b < a.T ? 1 : 0};
  const int first = min(max(fresh_index(a.cu + b), 0), a.T), end = min(fresh_index(a.cu + b + 1), a.T);
  return {first, max(end - first, 0)};
}
__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) {
  return min(max(fresh_index(a.lengths + b), 0), a.limit);
}
__device__ __forceinline__ int prefix_length(const PrefixArgs& a, int g) {
  return g < 0 ? 0 : min(max(fresh_index(a.prefix_lens + g), 0), a.prefix_limit);
}
// A request's group; -1: none, it has no prefix.
__device__ __forceinline__ int group_of(const PrefixArgs& a, int b) {
  if (!a.cu_groups) return a.G > 0 ? 0 : -1;
  int low = 0, high = a.G;                 // the first g whose end is behind b
  while (low < high) {
    const int mid = (low + high) >> 1;
    if (fresh_index(a.cu_groups + mid + 1) > b) high = mid;
    else low = mid + 1;
  }
  return low < a.G && fresh_index(a.cu_groups + low) <= b ? low : -1;
}
__device__ __forceinline__ int page_in(const PrefixArgs& a, int number) {
  return min(max(number, 0), a.pages - 1);
}

}  // namespace gf
