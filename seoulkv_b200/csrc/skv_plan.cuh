// skv_plan.cuh -- the list of key tiles that the attention operators work
// through, cut into contiguous ranges (items).
#pragma once
#include <cstdint>

namespace skv {

constexpr int PLAN_BATCH = 128;  // sequences of one launch (their tile counts are kept in shared memory)

// The list: sequence after sequence, unit (KV head) after unit, tile after
// tile; every unit ends with `idle` places that stand for its fixed cost.
struct Plan {
  long long total;  // places in the list
  int items;        // ranges that are not empty
  __device__ Plan(long long total_, int items_) : total(total_), items((int)min((long long)items_, total_)) {}
  __device__ long long begin(int i) const { return i < items ? quotient(total * i, items) : total; }
  // the item whose range holds place g
  __device__ int owner(long long g) const { return (int)quotient((g + 1) * items - 1, total); }
  // (a 64-bit division takes a few hundred cycles, and every role starts with some)
  static __device__ long long quotient(long long a, long long b) {
    return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
  }
};

// n / d for 0 <= n < 2^18 by a multiplication with ceil(2^32 / d), d <= 2^12.
__device__ __forceinline__ int by_inverse(int n, uint64_t inverse) { return (int)(((uint64_t)(uint32_t)n * inverse) >> 32); }

// pre[b] (places of the sequences before b, one unit's worth) and len[b], by
// one warp: KT cached tokens a tile, and `extra` places more.
template <int KT>
__device__ __forceinline__ void tile_prefix(const int32_t *lengths, int64_t stride, int t, int batch, int extra,
                                            int32_t *len, int32_t *pre) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const int b = b0 + lane;
    int n = 0, tiles = 0;
    if (b < batch) {
      n = __ldcg(lengths + b * stride);  // (from L2: k_tree_combine reads before it waits)
      n = max(0, min(n, t));
      tiles = (n + KT - 1) / KT + extra;
    }
    int x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (b < batch) {
      if (len) len[b] = n;
      pre[b + 1] = base + x;
    }
    base += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) pre[0] = 0;
}

// The segments of places [g, end): tiles [tile, tile + count) of one unit of
// `tiles`, at place `start`.
struct Walk {
  long long g, end, start = 0;
  const int32_t *pre;
  int units, idle;  // units per sequence
  int b = 0, unit = 0, tile = 0, count = 0, tiles = 0;
  __device__ Walk(const int32_t *pre_, int batch, int units_, int idle_, long long g_, long long end_)
      : g(g_), end(end_), pre(pre_), units(units_), idle(idle_) {
    int lo = 0, hi = batch - 1;  // the last sequence that starts at or before g
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)pre[mid] * units <= g) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  __device__ bool next() {
    while (g < end) {
      while ((long long)pre[b + 1] * units <= g) ++b;
      const int places = pre[b + 1] - pre[b];
      const long long rel = g - (long long)pre[b] * units;
      unit = (int)Plan::quotient(rel, places);
      tile = (int)(rel - (long long)unit * places);
      start = g - tile;
      tiles = places - idle;
      g = min(end, start + places);
      count = min(tiles, (int)(g - start)) - tile;
      if (count > 0) return true;
    }
    return false;
  }
};

}  // namespace skv
