// skv_evict.cu -- eviction from a cache by accumulated attention weight.
//
// Per (sequence, KV head) with n valid tokens and a budget of `keep`: the
// first `sink` and the last `local` tokens stay, and of the rest the
// keep - sink - local of largest weight (equal weights: the lowest index; NaN
// below every number).  n <= keep keeps everything.  The kept tokens' K, V
// and weights move to the front in their order; rows past them are zero,
// their ids -1.
//
// Two launches.  k_evict_select, one cluster per (sequence, head): the weights
// are mapped to integers of the same order, and up to four histogram passes of
// 8 bits find the value of the last kept one (fewer when a bin is kept whole);
// the ranks of the tokens above it and of the ties in index order give every
// kept token its place, so ids come out sorted and the result does not depend
// on the order of any atomic (they only count).  A pass is a few
// synchronisations of the cluster and one exchange of 1 KB per CTA: 256 bins,
// since an exchange of 2048 (three passes of 11 bits) took 3600 cycles each.
// k_evict_gather then moves the rows at copy bandwidth: every byte is read
// once and written once.
//
// Measured: 131072 tokens of 4 heads of 256 halved, BF16: 105.6 us, of which the
// gather of 537 MB takes 82 (6.5 TB/s, the copy rate) and the choice the rest;
// 5 requests of up to 4103 tokens in FP8: 17.7 us a call, the host's time (14.6
// us on the device).
#include <cooperative_groups.h>

#include "skv_ops.cuh"

namespace cg = cooperative_groups;

namespace skv {
namespace {

constexpr int EV_THREADS = 1024, EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 256;
// copies of the histogram, one per lane modulo 8: weights share exponents, so
// a warp's counts fall on few bins and one copy would serialise them
constexpr int EV_COPIES = 8;
constexpr int EV_CACHED = 49152;  // most keys that a CTA holds in shared memory (192 KB); longer segments are read again
constexpr int EV_CLUSTER = 16;    // most CTAs of a row
constexpr int EV_ROW = 2048;      // tokens of a row up to which one CTA is enough, and per CTA beyond

struct EvictArgs {
  const float *weights;
  int64_t ws[3];  // element strides (sequence, head, token)
  const int32_t *lengths;
  int64_t len_stride;
  int32_t *ids, *out_lengths;
  float *out_w;
  int heads, t, keep, sink, local;
  int room;  // keys that fit into the launch's shared memory
};

struct SelectSmem {
  uint32_t hist[EV_COPIES][EV_BINS];
  uint32_t sum[2][EV_BINS];
  uint32_t scan[EV_WARPS];
  uint32_t tie[EV_WARPS];
  uint32_t found[3];   // bin, still wanted inside it, its count
  uint32_t total[2];   // this CTA's kept-above and tied counts
};  // (keys follow)

// Larger weight, larger key; -0 equals +0, NaN is 0 (below -inf).
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

__global__ void __launch_bounds__(EV_THREADS) k_evict_select(EvictArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SelectSmem &s = *reinterpret_cast<SelectSmem *>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int row = blockIdx.x / ranks;
  const int b = row / a.heads, h = row - b * a.heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  grid_dependency_release();
  const int n = max(0, min(a.lengths[b * a.len_stride], a.t));
  const int m = min(n, a.keep);
  const float *w = a.weights + b * a.ws[0] + h * a.ws[1];
  int32_t *ids = a.ids + (int64_t)row * a.keep;
  float *out_w = a.out_w + (int64_t)row * a.keep;
  if (h == 0 && rank == 0 && tid == 0) a.out_lengths[b] = m;
  for (int j = m + rank * EV_THREADS + tid; j < a.keep; j += ranks * EV_THREADS) {
    ids[j] = -1;
    out_w[j] = 0.0f;
  }
  // a warp owns consecutive tokens, so that ballots give places in index order
  const int warps = ranks * EV_WARPS;
  const int seg = ((n + warps - 1) / warps + 31) & ~31;
  const int begin = min(n, (rank * EV_WARPS + warp) * seg), end = min(n, begin + seg);
  const bool cached = seg * EV_WARPS <= a.room;
  uint32_t *mine = reinterpret_cast<uint32_t *>(&s + 1) + (cached ? warp * seg : 0);
  const int lo = n <= a.keep ? n : a.sink, hi = n - a.local;  // the middle that competes: [lo, hi)
  auto key_at = [&](int i) { return cached ? mine[i - begin] : order_key(w[i * a.ws[2]]); };
  if (cached) {
#pragma unroll 4
    for (int i = begin + lane; i < end; i += 32) mine[i - begin] = order_key(w[i * a.ws[2]]);
  }
  uint32_t want = n <= a.keep ? 0u : (uint32_t)(a.keep - a.sink - a.local);
  uint32_t edge = 0xffffffffu;  // kept above it, ties in index order
  uint32_t ties = 0;
  if (want) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < EV_COPIES * EV_BINS; i += EV_THREADS) (&s.hist[0][0])[i] = 0;
      __syncthreads();
      uint32_t *hist = s.hist[lane % EV_COPIES];
#pragma unroll 4
      for (int i = begin + lane; i < end; i += 32) {
        const uint32_t k = key_at(i);
        if (i >= lo && i < hi && (shift == 24 || k >> (shift + 8) == prefix)) atomicAdd(hist + (k >> shift & 255u), 1u);
      }
      __syncthreads();
      uint32_t *sum = s.sum[shift >> 3 & 1];
      if (tid < EV_BINS) {
        uint32_t x = 0;
#pragma unroll
        for (int c = 0; c < EV_COPIES; ++c) x += s.hist[c][tid];
        sum[tid] = x;
      }
      // (also keeps the other buffer's remote readers of the pass before apart from its next writes)
      if (ranks > 1) cluster.sync(); else __syncthreads();
      // thread t: bin 255 - t, so that a prefix sum runs from the largest keys down
      uint32_t count = 0, inc = 0;
      if (tid < EV_BINS) {
        const int bin = EV_BINS - 1 - tid;
        for (int r = 0; r < ranks; ++r) count += ranks > 1 ? cluster.map_shared_rank(sum, r)[bin] : sum[bin];
        inc = warp_inclusive(count, lane);
        if (lane == 31) s.scan[warp] = inc;
      }
      __syncthreads();
      if (tid < EV_BINS) {
        for (int x = 0; x < warp; ++x) inc += s.scan[x];
        if (inc - count < want && want <= inc) {
          s.found[0] = (uint32_t)(EV_BINS - 1 - tid);
          s.found[1] = want - (inc - count);
          s.found[2] = count;
        }
      }
      __syncthreads();
      prefix = prefix << 8 | s.found[0];
      want = s.found[1];
      edge = prefix;
      ties = want;
      if (want == s.found[2] && prefix) {  // the bin is kept whole: everything from its first key on
        edge = (prefix << shift) - 1;
        ties = 0;
        break;
      }
    }
  }
  // places: tokens kept for certain and tied ones, counted per warp, CTA and cluster
  auto kinds = [&](int i, bool &above, bool &tied) {
    above = tied = false;
    if (i >= end) return;
    if (i < lo || i >= hi) {
      above = true;
    } else {
      const uint32_t k = key_at(i);
      above = k > edge;
      tied = ties && k == edge;
    }
  };
  uint32_t n_above = 0, n_tied = 0;
  __syncwarp();
#pragma unroll 4
  for (int i0 = begin; i0 < end; i0 += 32) {
    bool above, tied;
    kinds(i0 + lane, above, tied);
    n_above += __popc(__ballot_sync(0xffffffffu, above));
    n_tied += __popc(__ballot_sync(0xffffffffu, tied));
  }
  if (lane == 0) s.scan[warp] = n_above, s.tie[warp] = n_tied;
  __syncthreads();
  if (warp == 0) {
    const uint32_t x = warp_inclusive(s.scan[lane], lane), y = warp_inclusive(s.tie[lane], lane);
    s.scan[lane] = x;
    s.tie[lane] = y;
    if (lane == 31) s.total[0] = x, s.total[1] = y;
  }
  __syncthreads();
  if (ranks > 1) cluster.sync();
  uint32_t at = warp ? s.scan[warp - 1] : 0u, tie = warp ? s.tie[warp - 1] : 0u;
  for (int r = 0; r < rank; ++r) {
    const uint32_t *o = cluster.map_shared_rank(s.total, r);
    at += o[0];
    tie += o[1];
  }
  const uint32_t below = (1u << lane) - 1u;
  constexpr int BLOCKS = 4;  // of 32 tokens, whose weights are loaded together
  for (int i0 = begin; i0 < end; i0 += 32 * BLOCKS) {
    float x[BLOCKS];
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      const int i = i0 + 32 * u + lane;
      x[u] = i < end ? w[i * a.ws[2]] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      bool above, tied;
      const int i = i0 + 32 * u + lane;
      kinds(i, above, tied);
      const uint32_t ba = __ballot_sync(0xffffffffu, above), bt = __ballot_sync(0xffffffffu, tied);
      const uint32_t tie_before = tie + __popc(bt & below);
      if (above || (tied && tie_before < ties)) {
        const uint32_t place = at + __popc(ba & below) + min(tie_before, ties);
        ids[place] = i;
        out_w[place] = x[u];
      }
      at += __popc(ba);
      tie += __popc(bt);
    }
  }
  if (ranks > 1) cluster.sync();  // no CTA leaves while another reads its counts
}

constexpr int EG_THREADS = 256, EG_ROWS = 4;  // rows whose K and V loads one thread has in flight

struct GatherArgs {
  const uint8_t *x[2];
  uint8_t *y[2];
  int64_t xs[2][3];  // byte strides (sequence, head, token)
  const int32_t *ids;
  int64_t rows;
  int heads, keep, row_bytes;
};

template <typename C>
__global__ void __launch_bounds__(EG_THREADS) k_evict_gather(GatherArgs a) {
  const int per_row = a.row_bytes / (int)sizeof(C);
  const int lanes = min(per_row, EG_THREADS), group = EG_THREADS / lanes;
  const int mine = threadIdx.x / lanes;
  if (mine >= group) return;  // (no barrier below)
  grid_dependency_wait();
  grid_dependency_release();
  const int64_t row0 = (int64_t)blockIdx.x * group * EG_ROWS + mine;
  for (int c = threadIdx.x - mine * lanes; c < per_row; c += lanes) {
    C v[EG_ROWS][2];
    int32_t id[EG_ROWS];
#pragma unroll
    for (int u = 0; u < EG_ROWS; ++u) {
      const int64_t r = row0 + u * group;
      id[u] = r < a.rows ? a.ids[r] : -1;
    }
#pragma unroll
    for (int u = 0; u < EG_ROWS; ++u) {
      v[u][0] = v[u][1] = C{};
      if (id[u] < 0) continue;
      const int64_t bh = (row0 + u * group) / a.keep;
      const int b = (int)(bh / a.heads), h = (int)(bh - (int64_t)b * a.heads);
#pragma unroll
      for (int w = 0; w < 2; ++w)
        v[u][w] = __ldcs(reinterpret_cast<const C *>(a.x[w] + b * a.xs[w][0] + h * a.xs[w][1] + id[u] * a.xs[w][2]) + c);
    }
#pragma unroll
    for (int u = 0; u < EG_ROWS; ++u) {
      const int64_t r = row0 + u * group;
      if (r >= a.rows) break;
#pragma unroll
      for (int w = 0; w < 2; ++w) __stcs(reinterpret_cast<C *>(a.y[w] + r * a.row_bytes) + c, v[u][w]);
    }
  }
}

template <typename C>
cudaError_t launch_gather(const GatherArgs &g, cudaStream_t st) {
  const int per_row = g.row_bytes / (int)sizeof(C);
  const int group = EG_THREADS / (per_row < EG_THREADS ? per_row : EG_THREADS);
  const int64_t blocks = (g.rows + group * EG_ROWS - 1) / (group * EG_ROWS);
  return op_launch(k_evict_gather<C>, dim3((unsigned)blocks), dim3(EG_THREADS), 0, st, 1, g);
}

}  // namespace
}  // namespace skv

extern "C" int skv_evict(const SkvEvict *d, void *stream) {
  using namespace skv;
  if (!d) return op_fail(SKV_E_INVALID, "null descriptor");
  if (d->batch < 0 || d->kv_heads < 1 || d->tokens < 1 || d->tokens > INT32_MAX / 2 || d->dim < 1 || d->dim > 65536 ||
      (d->element_bytes != 1 && d->element_bytes != 2 && d->element_bytes != 4) || d->batch > (1 << 24) ||
      d->kv_heads > (1 << 24) || d->batch * d->kv_heads > (1 << 24))
    return op_fail(SKV_E_INVALID, "batch, heads, tokens, dim or element_bytes out of range");
  if (d->keep < 1 || d->keep > d->tokens || d->sink < 0 || d->local < 0 || d->sink > d->keep || d->local > d->keep - d->sink)
    return op_fail(SKV_E_INVALID, "keep must be in [1, tokens] and hold the sink and local tokens");
  const int64_t rows = d->batch * d->kv_heads * d->keep;
  if (rows > (int64_t)INT32_MAX * 8) return op_fail(SKV_E_INVALID, "too many kept rows");
  if (d->batch == 0) return SKV_OK;
  if (!d->k || !d->v || !d->weights || !d->lengths || !d->k_out || !d->v_out || !d->weights_out || !d->ids || !d->lengths_out)
    return op_fail(SKV_E_INVALID, "null input or output pointer");
  if (d->dim > 1 && (d->k_stride[3] != 1 || d->v_stride[3] != 1))
    return op_fail(SKV_E_INVALID, "the innermost dimension must be contiguous");
  int sms = 0;
  if (int rc = sm_count(d->device, &sms)) return rc;
  DeviceScope scope((int)d->device);
  if (int rc = op_cuda(scope.error(), "selecting the device")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  EvictArgs a;
  a.weights = static_cast<const float *>(d->weights);
  const int64_t size[3] = {d->batch, d->kv_heads, d->tokens};
  op_strides(a.ws, d->weights_stride, size, 3);
  op_strides(&a.len_stride, &d->lengths_stride, size, 1);
  a.lengths = static_cast<const int32_t *>(d->lengths);
  a.ids = static_cast<int32_t *>(d->ids);
  a.out_lengths = static_cast<int32_t *>(d->lengths_out);
  a.out_w = static_cast<float *>(d->weights_out);
  a.heads = (int)d->kv_heads, a.t = (int)d->tokens, a.keep = (int)d->keep;
  a.sink = (int)d->sink, a.local = (int)d->local;
  static bool set[64], wide[64];
  int rc = SKV_OK;
  if (!__atomic_load_n(&wide[d->device], __ATOMIC_RELAXED)) {  // clusters of 16 are not portable
    rc = op_cuda(cudaFuncSetAttribute(k_evict_select, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cluster size");
    if (!rc) __atomic_store_n(&wide[d->device], true, __ATOMIC_RELAXED);
  }
  if (!rc) rc = op_shared_memory(reinterpret_cast<const void *>(&k_evict_select), (int)sizeof(SelectSmem) + EV_CACHED * 4, (int)d->device, set);
  if (rc) return rc;
  // CTAs of a row: as many as its length gives work to, while all rows fit on
  // the device together.  Measured (with a gather of almost nothing), one CTA
  // a row and up to sixteen: 4 rows of 4103 tokens 13.7 and 13.0 us, of 16384
  // 23.0 and 15.8, of 131072 213 and 27.4.
  int ranks = 1;
  while (ranks < EV_CLUSTER && d->tokens > (int64_t)EV_ROW * ranks && d->batch * d->kv_heads * ranks * 2 <= sms) ranks *= 2;
  const int64_t warps = (int64_t)ranks * EV_WARPS, keys = ((d->tokens + warps - 1) / warps + 31) / 32 * 32 * EV_WARPS;
  a.room = keys <= EV_CACHED ? (int)keys : 0;
  rc = op_cuda(op_launch(k_evict_select, dim3((unsigned)(d->batch * d->kv_heads * ranks)), dim3(EV_THREADS),
                         sizeof(SelectSmem) + (size_t)a.room * 4, st, (unsigned)ranks, a), "k_evict_select launch");
  if (rc) return rc;
  GatherArgs g;
  g.x[0] = static_cast<const uint8_t *>(d->k), g.x[1] = static_cast<const uint8_t *>(d->v);
  g.y[0] = static_cast<uint8_t *>(d->k_out), g.y[1] = static_cast<uint8_t *>(d->v_out);
  g.row_bytes = (int)(d->dim * d->element_bytes);
  uintptr_t all = (uintptr_t)g.x[0] | (uintptr_t)g.x[1] | (uintptr_t)g.y[0] | (uintptr_t)g.y[1] | (uintptr_t)g.row_bytes;
  op_strides(g.xs[0], d->k_stride, size, 3);
  op_strides(g.xs[1], d->v_stride, size, 3);
  for (int i = 0; i < 3; ++i) {
    g.xs[0][i] *= d->element_bytes, g.xs[1][i] *= d->element_bytes;
    all |= (uintptr_t)g.xs[0][i] | (uintptr_t)g.xs[1][i];
  }
  g.ids = a.ids;
  g.rows = rows;
  g.heads = a.heads, g.keep = a.keep;
  // the widest access that every row start allows
  cudaError_t e = all % 16 == 0  ? launch_gather<uint4>(g, st)
                  : all % 4 == 0 ? launch_gather<uint32_t>(g, st)
                  : all % 2 == 0 ? launch_gather<uint16_t>(g, st)
                                 : launch_gather<uint8_t>(g, st);
  return op_cuda(e, "k_evict_gather launch");
}
