// skv_tree.cu -- exact attention of a tree of drafted tokens over a cache.
//
// N <= 64 drafted tokens (nodes) of one sequence see its cache and their own
// ancestors.  With G query heads per KV head, one KV head has R = N * G rows
// (row r: node r / G, query head r % G) over one stream of keys: the cache's
// tiles, then one tile of the N nodes' own keys under the ancestor mask.
//   s = scale q.k,  out = sum exp(s - m) v / sum exp(s - m),  lse = m + log sum exp(s - m)
// in one pass with a running maximum; the row statistics and the accumulator
// are FP32 (the accumulator in tensor memory).
//
// Both products run on tcgen05 with the rows as M = 128 lanes: S = Q K^T with
// Q in shared memory (64 KB at D = 256; tensor memory is full: O has 256
// columns, two score tiles 128 each), and O += P V with P = exp(s - m) written
// over S as BF16, rounded once (at most 2^-8 of each weight; the row sum is
// taken before rounding).  Tiles are 128 keys: an MMA of N = 64 takes as long
// as one of N = 128.  K and V arrive by TMA in a ring of 160 KB and more per
// SM, which is what carries the HBM bandwidth.
//
// Two threads per row do the softmax, each half of a tile's columns.  The
// scores of tile g + 1 are computed beside the softmax of tile g.  The maximum
// moves only when it grows by more than 2^8, so that O is hardly ever scaled.
//
// Over an FP8 cache K goes to the tensor core as it is stored, against queries
// split into two FP8 rows (skv_tensor.cuh); V is turned into BF16 by four
// groups of two warps, since FP8 weights would lose the tail of a softmax.
//
// The tiles of all units (sequence, KV head, 128 rows) form one list that is
// cut into equal contiguous ranges, one per CTA (one CTA per SM): ragged
// lengths balance by themselves.  A unit that one CTA covers is written at
// once; of a unit cut across CTAs every CTA writes its partial (m, l, O) and
// k_tree_combine joins them in order, so that results do not depend on timing.
// The cut is worked out on the device from the lengths: no host wait, and a
// captured graph follows its caches as they grow.  (Ranges handed out as CTAs
// become free were slower: 94 -> 99 us for the token below, 208 -> 212 for the
// requests, since the fixed ranges already read at the copy rate.)  Short
// caches are not cut at all (tree_whole).
//
// What bounds it, measured at 16 query heads on 4 KV heads of 256 (a copy
// moves 6437 GB/s):
// (in long loops, where the power cap lowers the clock to 1.1 to 1.6 GHz; in
// brackets at 1965 MHz)
//   one token, 131072 cached, BF16: 92 us (86), 537 MB = 91% of the copy rate
//     (more tokens add bytes at 7.2 TB/s; starting and joining 148 partials are
//     a fixed 14 us);
//   64 nodes (256 rows a KV head): 163 us (141; one cache again and again 129).
//     138 GFLOP would take 102 us at the 1349 TFLOP/s that the clock under load
//     sustains; the tensor pipe is busy 70% of the active cycles, and the
//     softmax of 268M scores beside it is what keeps it waiting;
//   16 requests of up to 32768, 12 nodes: 200 us (190), 1.08 GB = 84%;
//   8 nodes over an FP8 cache of 131072: 82 us (69), 269 MB = 51% (more tokens
//     add bytes at 4.1 to 4.8 TB/s).  No pipe is half full: DRAM 43%, tensor
//     43%, ALU 33%, shared memory 34%.  The chain of a V stage (load,
//     conversion, product) bounds it, since a converting group has one place
//     before and one behind its conversion at D = 256.  A shorter conversion
//     shortens the chain; without any, a tile takes a sixth less.  The second
//     half of the queries and the exponentials cost nothing;
//   3 ragged caches of up to 327, 5 nodes: 13 us a call, the host's time (12 us
//     on the device).
#include <cuda_bf16.h>

#include <mutex>

#include "skv_device.cuh"
#include "skv_exchange.cuh"
#include "skv_ops.cuh"
#include "skv_plan.cuh"
#include "skv_tensor.cuh"
#include "skv_tree.cuh"

namespace skv {

__device__ uint32_t g_op_status;

int status_word(int device, uint32_t **word) {
  static std::mutex lock;
  static uint32_t *known[64] = {};
  if (device < 0 || device >= 64) return op_fail(SKV_E_INVALID, "device ordinal out of range");
  std::lock_guard<std::mutex> hold(lock);
  if (!known[device]) {
    void *p = nullptr;
    if (int rc = op_cuda(cudaGetSymbolAddress(&p, g_op_status), "cudaGetSymbolAddress(status)")) return rc;
    known[device] = static_cast<uint32_t *>(p);
  }
  *word = known[device];
  return SKV_OK;
}

namespace {

using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                            const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
  static const Encode encode = [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  return encode;
}

}  // namespace

int make_map(CUtensorMap *map, const void *base, int64_t dim, int64_t rows, int64_t ny, int64_t nz,
             const int64_t *stride, int box_rows, int pieces) {
  const Encode encode = encoder();
  if (!encode) return op_fail(SKV_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const int64_t n[3] = {rows, ny, nz};
  cuuint64_t size[5] = {64, 1, (cuuint64_t)dim / 64, 1, 1}, step[4] = {0, 128, 0, 0};
  for (int i = 0; i < 3; ++i) {
    const bool one = n[i] == 1 || stride[i] == 0;
    const int at = i ? i + 2 : 1;
    size[at] = one ? 1 : (cuuint64_t)n[i];
    step[at - 1] = one ? (cuuint64_t)dim * 2 : (cuuint64_t)stride[i] * 2;
  }
  const cuuint32_t box[5] = {64, (cuuint32_t)box_rows, (cuuint32_t)pieces, 1, 1}, unit[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void *>(base), size, step, box, unit,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SKV_OK : op_fail(SKV_E_INVALID, "cuTensorMapEncodeTiled: error %d", (int)r);
}

int make_byte_map(CUtensorMap *map, const void *base, int64_t bytes, int64_t rows, int64_t ny, int64_t nz,
                  const int64_t *stride, int box_rows, int box_bytes, bool swizzle) {
  const Encode encode = encoder();
  if (!encode) return op_fail(SKV_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const int64_t n[3] = {rows, ny, nz};
  cuuint64_t size[4] = {(cuuint64_t)bytes, 1, 1, 1}, step[3];
  for (int i = 0; i < 3; ++i) {
    const bool one = n[i] == 1 || stride[i] == 0;
    size[i + 1] = one ? 1 : (cuuint64_t)n[i];
    step[i] = one ? (cuuint64_t)bytes : (cuuint64_t)stride[i];
  }
  const cuuint32_t box[4] = {(cuuint32_t)box_bytes, (cuuint32_t)box_rows, 1, 1}, unit[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void *>(base), size, step, box, unit,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            !swizzle           ? CU_TENSOR_MAP_SWIZZLE_NONE
                            : box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                               : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SKV_OK : op_fail(SKV_E_INVALID, "cuTensorMapEncodeTiled: error %d", (int)r);
}

namespace {

constexpr int TR_NODES = SKV_TREE_MAX_NODES;
constexpr int TR_KEYS = 128;   // keys of a tile
constexpr int TR_ROWS = 128;   // rows of a unit: the MMA's M
constexpr int TR_GROUP = 64;   // threads that turn an FP8 stage into BF16
constexpr int TR_IDLE = 1;     // what starting and ending a unit costs, in tiles
constexpr int TR_JOIN = 5;     // what cutting units and joining their parts costs, in tiles

template <int D_, bool F8_>
struct TreeCfg {
  static constexpr int D = D_;
  static constexpr bool F8 = F8_;
  static constexpr int KT = TR_KEYS;
  static constexpr int PIECES = D / 64;   // ring stages of a BF16 tile of K or V
  static constexpr int VROWS = KT / PIECES;  // keys of a V stage
  static constexpr int STAGE = KT * 128;  // bytes: K 128 keys x 64 dimensions, V VROWS keys x D
  // FP8: K tiles as they are stored in a ring of their own (128 or 64 bytes of
  // every key a stage), V before its conversion in another.  The rings of V
  // are multiples of the converting groups, so that a place in them belongs to
  // one group, which sees its phases in turn.
  static constexpr int ROW8 = D < 128 ? D : 128, PIECES8 = D / ROW8;
  static constexpr int NK8 = F8 ? 4 : 0;
  static constexpr int RAW = STAGE / 2;
  static constexpr int NRAW = F8 ? (D == 256 ? 4 : 8) : 0;
  static constexpr int NSTAGE = F8 ? 4 : D == 256 ? 10 : D == 128 ? 11 : 12;
  static constexpr int THREADS = F8 ? 576 : 384;  // FP8: warps 2, 3 and 12.. convert
  static constexpr int COL_S = 256;       // tensor memory columns: O, then two score tiles (P over S)
  static constexpr int QBYTES = TR_ROWS * D * 2;  // BF16, or both FP8 halves
  static constexpr int RING = QBYTES + (NSTAGE + NK8) * STAGE + NRAW * RAW;
};

struct TreeMaps {
  CUtensorMap k, v, kn, vn;  // cache and nodes
};

struct TreeArgs {
  const uint16_t *q;
  int64_t qs[3];  // element strides (sequence, node, head)
  const CUtensorMap *cell_maps;  // FP8 caches in separate buffers: K and V maps of cell = sequence * heads + head
  const uint16_t *kn, *vn;
  int64_t kns[3], vns[3];  // element strides (sequence, head, node)
  const int32_t *lengths;
  int64_t len_stride;
  const int32_t *parents;
  int64_t ps[2];           // element strides (sequence, node)
  uint16_t *out;           // [sequence][node][query head][D]
  float *lse;              // [sequence][node][query head]
  float2 *ml;              // partials: [slot][rows] (m in log2 units, l; l < 0: the row is unused)
  float *part;             // [slot][rows][D]
  uint64_t by_group;       // (by_inverse)
  int32_t batch, n, heads, group, t, mtiles, rows;
  int32_t whole;           // an item is a unit, and nothing is left to join
  int32_t along[4][2];     // coordinate steps (head, sequence) of the four maps: 0 where one element stands for all
  float c2;                // scale * log2(e)
  uint32_t *status;
};

template <class C>
struct TreeSmem {
  uint64_t full[C::NSTAGE], empty[C::NSTAGE];
  uint64_t raw_full[C::F8 ? C::NRAW : 1], raw_empty[C::F8 ? C::NRAW : 1];
  uint64_t k8_full[C::F8 ? C::NK8 : 1], k8_empty[C::F8 ? C::NK8 : 1];
  float scale2[C::F8 ? TR_ROWS : 1];  // of the split queries' rows: scale * log2(e), by the row's power of two
  uint64_t q_ready, s_full[2], p_ready[2], o_done[2], drain;
  uint64_t anc[TR_NODES];      // nodes that node i sees (0: unused)
  unsigned long long bad;      // nodes with a value that is not finite
  float share[2][TR_ROWS];     // maxima and sums that the two threads of a row exchange (exchange_slot)
  int8_t up[TR_NODES];         // the node before (-1: the cache, -2: none, unused)
  uint32_t tmem;
  uint32_t abort;
  int32_t pre[PLAN_BATCH + 1];  // places of the sequences before (one unit's worth)
};

// Order of a segment's 2n operand tiles: K0, K1, V0, K2, V1, ..., V(n-1), the
// order in which the tensor core needs them.
__device__ __forceinline__ int pos_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }
__device__ __forceinline__ void tile_at(int p, int n, bool &is_v, int &i) {
  is_v = p == 2 * n - 1 || (p > 0 && !(p & 1));
  i = p == 0 ? 0 : p == 2 * n - 1 ? n - 1 : is_v ? (p - 2) / 2 : (p + 1) / 2;
}
// Over an FP8 cache the BF16 ring has the V tiles and the nodes' K: a segment
// with the nodes (in its last tile) has n + 1 tiles there, the nodes' K at
// this place among them.
__device__ __forceinline__ int nodes_k_place(int n) { return n > 1 ? n - 2 : 0; }

__device__ __forceinline__ bool not_finite_bf16(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }

// ---- the attention kernel ----------------------------------------------------

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    k_tree_attention(const __grid_constant__ TreeMaps maps, const __grid_constant__ TreeArgs a) {
  constexpr int D = C::D, KT = C::KT;
  extern __shared__ __align__(1024) uint8_t smem_dyn[];
  uint8_t *queries = smem_dyn;  // [D / 64][128 rows][128 bytes], swizzled
  uint8_t *ring = queries + C::QBYTES;
  uint8_t *ring8 = ring + C::NSTAGE * C::STAGE, *raw = ring8 + C::NK8 * C::STAGE;
  TreeSmem<C> &s = *reinterpret_cast<TreeSmem<C> *>(smem_dyn + C::RING);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (warp == 0) {
    if (lane == 0) {
      if (!a.cell_maps) {
        tma_prefetch_map(&maps.k);
        tma_prefetch_map(&maps.v);
      }
      if (!C::F8) {
        tma_prefetch_map(&maps.kn);
        tma_prefetch_map(&maps.vn);
      }
    }
    grid_dependency_wait();
    tile_prefix<KT>(a.lengths, a.len_stride, a.t, a.batch, 1 + TR_IDLE, nullptr, s.pre);
  } else if (warp == 1) {
    tmem_alloc(&s.tmem, 512);
  } else if (warp == 2 && lane == 0) {
    for (int i = 0; i < C::NSTAGE; ++i) {
      bar_init(&s.full[i], C::F8 ? TR_GROUP / 32 : 1);
      bar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < C::NRAW; ++i) {
      bar_init(&s.raw_full[i], 1);
      bar_init(&s.raw_empty[i], TR_GROUP / 32);
    }
    for (int i = 0; i < C::NK8; ++i) {
      bar_init(&s.k8_full[i], 1);
      bar_init(&s.k8_empty[i], 1);
    }
    bar_init(&s.q_ready, 8);
    bar_init(&s.drain, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(&s.s_full[i], 1);
      bar_init(&s.p_ready[i], 8);
      bar_init(&s.o_done[i], 1);
    }
    bar_init_fence();
    s.abort = 0;
    s.bad = 0;
  }
  grid_dependency_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_release();
  const uint32_t tmem = *(volatile uint32_t *)&s.tmem;
  volatile uint32_t *abort = &s.abort;
  // CTA: item (blockIdx / mtiles) of the list for one 128-row part of its
  // units; the parts of an item are neighbours, so that they read the same
  // keys at the same time and HBM delivers them once
  const Plan plan((long long)s.pre[a.batch] * a.heads, (int)gridDim.x / a.mtiles);
  const int item = blockIdx.x / a.mtiles, mt = blockIdx.x % a.mtiles;
  long long from = 0, to = 0;
  if (a.whole) {
    const int b = item / a.heads, places = s.pre[b + 1] - s.pre[b];
    from = (long long)s.pre[b] * a.heads + (long long)(item - b * a.heads) * places, to = from + places;
  } else {
    from = plan.begin(item), to = plan.begin(item + 1);
  }
  const Walk walk(s.pre, a.batch, a.heads, TR_IDLE, from, to);
  auto wait = [&](uint64_t *bar, uint32_t parity) { return bar_wait(bar, parity, abort, a.status); };
  auto length = [&](int b) { return max(0, min(a.lengths[b * a.len_stride], a.t)); };

  if (warp == 0) {
    // ---- loads: BF16 tiles into the ring; of FP8 caches K into its own, and V
    // beside it to be converted
    const uint32_t one = elect_lane();
    Walk w = walk;
    uint32_t seq = 0, seq8 = 0;  // stages of the ring (or V stages before conversion), FP8 K stages
    bool ok = true;
    while (ok && w.next()) {
      const CUtensorMap *cell = C::F8 && a.cell_maps ? a.cell_maps + 2 * ((int64_t)w.b * a.heads + w.unit) : nullptr;
      if (cell) {
        tma_acquire_map(one, cell);
        tma_acquire_map(one, cell + 1);
      }
      for (int p = 0; ok && p < 2 * w.count; ++p) {
        bool is_v;
        int i;
        tile_at(p, w.count, is_v, i);
        const bool nodes = w.tile + i == w.tiles - 1;
        const int which = (nodes ? 2 : 0) + (is_v ? 1 : 0);
        const CUtensorMap *map = nodes ? (is_v ? &maps.vn : &maps.kn) : (is_v ? &maps.v : &maps.k);
        if (cell) map = cell + is_v;
        const int row = nodes ? 0 : (w.tile + i) * KT;
        const int y = w.unit * a.along[which][0], z = w.b * a.along[which][1];
        if constexpr (C::F8) {
          if (!nodes && !is_v) {
            for (int piece = 0; piece < C::PIECES8; ++piece, ++seq8) {
              const uint32_t slot = seq8 % C::NK8;
              if (!(ok = wait(&s.k8_empty[slot], ((seq8 / C::NK8) & 1) ^ 1))) break;
              tma_load_bytes(one, ring8 + slot * C::STAGE, map, piece * C::ROW8, row, y, z, &s.k8_full[slot], KT * C::ROW8);
            }
          } else {
            for (int piece = 0; piece < C::PIECES; ++piece, ++seq) {
              const uint32_t slot = seq % C::NRAW;
              if (!(ok = wait(&s.raw_empty[slot], ((seq / C::NRAW) & 1) ^ 1))) break;
              if (!nodes)
                tma_load_bytes(one, raw + slot * C::RAW, map, 0, row + piece * C::VROWS, y, z, &s.raw_full[slot], C::RAW);
              else if (one)  // (the converting warps copy the nodes: the place passes)
                bar_arrive(&s.raw_full[slot]);
            }
          }
        } else {
          for (int piece = 0; piece < C::PIECES; ++piece, ++seq) {
            const uint32_t slot = seq % C::NSTAGE;
            if (!(ok = wait(&s.empty[slot], ((seq / C::NSTAGE) & 1) ^ 1))) break;
            tma_load(one, ring + slot * C::STAGE, map, row + (is_v ? piece * C::VROWS : 0), is_v ? 0 : piece, y, z,
                     &s.full[slot], C::STAGE);
          }
        }
      }
    }
    if (!ok) {  // gave up: the copies in flight still land before the CTA ends
      const unsigned long long t0 = timer_ns();
      auto landed = [&](uint64_t *bar, uint32_t slots, uint32_t n) {
        for (uint32_t back = 1; back <= slots && back <= n; ++back)
          while (!bar_try(&bar[(n - back) % slots], ((n - back) / slots) & 1) && timer_ns() - t0 < WAIT_NS / 2) {
          }
      };
      if constexpr (C::F8) {
        landed(s.raw_full, C::NRAW, seq);
        landed(s.k8_full, C::NK8, seq8);
      } else {
        landed(s.full, C::NSTAGE, seq);
      }
    }
  } else if (warp == 1) {
    // ---- tensor core
    const uint32_t one = elect_lane();
    Walk w = walk;
    constexpr uint32_t DESC_S = mma_desc(TR_ROWS, KT, false), DESC_O = mma_desc(TR_ROWS, D, true);
    constexpr uint32_t DESC_S8 = mma_desc_f8(TR_ROWS, KT);
    const uint32_t q0 = s_addr(queries), ring0 = s_addr(ring), ring80 = s_addr(ring8);
    uint32_t seq = 0, seq8 = 0, gt = 0, loaded = 0;  // loaded: times that the queries were
    while (w.next()) {
      const int n = w.count;
      auto scores = [&](int i, uint32_t buf) {
        const uint32_t d = tmem + C::COL_S + buf * KT;
        if (C::F8 && w.tile + i < w.tiles - 1) {
#pragma unroll
          for (int piece = 0; piece < C::PIECES8; ++piece, ++seq8) {
            const uint32_t slot = seq8 % (C::F8 ? C::NK8 : 1);
            wait(&s.k8_full[slot], (seq8 / (C::F8 ? C::NK8 : 1)) & 1);
            const uint32_t k0 = ring80 + slot * C::STAGE, qp = q0 + piece * TR_ROWS * C::ROW8;
#pragma unroll
            for (int ks = 0; ks < C::ROW8 / 32; ++ks) {
              const uint64_t kd = smem_desc_rows(k0 + ks * 32, C::ROW8);
              mma_f8(one, d, smem_desc_rows(qp + ks * 32, C::ROW8), kd, DESC_S8, piece + ks > 0);
              mma_f8(one, d, smem_desc_rows(qp + TR_ROWS * D + ks * 32, C::ROW8), kd, DESC_S8, true);
            }
            mma_commit(one, &s.k8_empty[slot]);
          }
        } else {
          if (C::F8 && i > 0) wait(&s.q_ready, loaded++ & 1);  // the queries in BF16
#pragma unroll
          for (int piece = 0; piece < C::PIECES; ++piece, ++seq) {
            const uint32_t stage = seq % C::NSTAGE;
            wait(&s.full[stage], (seq / C::NSTAGE) & 1);
            const uint32_t k0 = ring0 + stage * C::STAGE, qp = q0 + piece * TR_ROWS * 128;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_ss(one, d, smem_desc(qp + ks * 32, 16), smem_desc(k0 + ks * 32, 16), DESC_S, piece + ks > 0);
            mma_commit(one, &s.empty[stage]);
          }
        }
        mma_commit(one, &s.s_full[buf]);
      };
      wait(&s.q_ready, loaded++ & 1);
      scores(0, gt & 1);
      for (int i = 0; i < n; ++i, ++gt) {
        const uint32_t buf = gt & 1;
        if (i + 1 < n) scores(i + 1, buf ^ 1);
        wait(&s.p_ready[buf], (gt >> 1) & 1);
        tc_fence_after();
#pragma unroll
        for (int piece = 0; piece < C::PIECES; ++piece, ++seq) {
          const uint32_t stage = seq % C::NSTAGE;
          wait(&s.full[stage], (seq / C::NSTAGE) & 1);
          const uint32_t v0 = ring0 + stage * C::STAGE, p0 = tmem + C::COL_S + buf * KT;
#pragma unroll
          for (int ks = 0; ks < C::VROWS / 16; ++ks) {
            const int key = piece * C::VROWS + 16 * ks;  // P of keys 64.. starts at column 64
            mma_ts(one, tmem, p0 + key / 64 * 64 + key % 64 / 2, smem_desc(v0 + ks * 2048, C::VROWS * 128), DESC_O,
                   i > 0 || key > 0);
          }
          mma_commit(one, &s.empty[stage]);
        }
        mma_commit(one, &s.o_done[buf]);
      }
    }
    if (*abort) {  // what was issued ends before tensor memory is given back
      mma_commit(one, &s.drain);
      const unsigned long long t0 = timer_ns();
      while (!bar_try(&s.drain, 0) && timer_ns() - t0 < WAIT_NS / 4) {
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // ---- softmax: two threads per row, each half of a tile's columns and of O's
    const int st = tid - 128, half = st >> 7, row = st & 127;
    const int pair = 2 + ((warp - 4) & 3);  // barrier of the two warps that share 32 rows
    const uint32_t lanes = tmem + ((uint32_t)((warp - 4) & 3) << 21);  // these 32 lanes (bits 16..)
    const int left = a.n * a.group - mt * TR_ROWS;  // rows of this part
    const bool warp_on = (row & ~31) < left, on = row < left;
    const int r = mt * TR_ROWS + row;  // row of the KV head
    const int node = on ? by_inverse(r, a.by_group) : 0, qg = on ? r - node * a.group : 0;
    // rows that do not exist are zeros: a product of zeros draws no power,
    // and power is what the clock follows
    for (int x = st; x < (TR_ROWS - min(left, TR_ROWS)) * (D / 8); x += 256) {
      const int at = min(left, TR_ROWS) + x / (D / 8), c16 = x % (D / 8);
      *reinterpret_cast<uint4 *>(queries + (c16 / 8) * TR_ROWS * 128 + at * 128 + (c16 % 8) * 16) = make_uint4(0, 0, 0, 0);
    }
    Walk w = walk;
    uint32_t base = 0, gt = 0;
    // Tile g's S and O.  Both alternate between two barriers, and S(g) follows
    // O(g - 2): a wait is never two phases behind, so its parity names one.
    auto done = [&](uint64_t *two, uint32_t g) {
      wait(&two[g & 1], (g >> 1) & 1);
      __syncwarp();
      tc_fence_after();
    };
    // The rows' queries of a unit: BF16, or (FP8 cache) split into two FP8 rows
    // whose sum they are.  Short loops: code that runs once per segment waits
    // for its instructions when it is unrolled.
    const int total = min(left, TR_ROWS) * (D / 8);
    auto row_at = [&](const Walk &x, int c) {  // the row that holds 16-byte piece c
      const int rr = mt * TR_ROWS + c / (D / 8), nd = by_inverse(rr, a.by_group);
      return a.q + x.b * a.qs[0] + nd * a.qs[1] + (x.unit * a.group + rr - nd * a.group) * a.qs[2] + c % (D / 8) * 8;
    };
    auto load_bf16 = [&](const Walk &x) {
#pragma unroll 1
      for (int c = st; c < total; c += 256) {
        const int at = c / (D / 8), c16 = c % (D / 8);
        cp_async16(queries + (c16 / 8) * TR_ROWS * 128 + at * 128 + ((c16 % 8) ^ (at & 7)) * 16, row_at(x, c), true);
      }
      cp_async_wait();
      async_fence();
      __syncwarp();
      if (lane == 0) bar_arrive(&s.q_ready);
    };
    auto load_split = [&](const Walk &x) {
      const int c16 = st % (D / 8);
      auto fetch = [&](int c) { return c < total ? __ldg(reinterpret_cast<const uint4 *>(row_at(x, c))) : make_uint4(0, 0, 0, 0); };
      // (whole warps, since a row's threads look at one another's)
      const int whole_warps = (total + 31) & ~31;
      uint4 ahead = fetch(st);
#pragma unroll 1
      for (int c = st; c < whole_warps; c += 256) {
        const uint4 v = ahead;
        ahead = fetch(c + 256);
        const int at = c / (D / 8);
        const uint32_t e = split_exponent(v, D / 8);
        uint2 hi, lo;
        split_eight(v, __uint_as_float(e << 23), hi, lo);
        uint8_t *to = queries + (c16 * 8 / C::ROW8) * TR_ROWS * C::ROW8 + at * C::ROW8 +
                      swizzled(c16 * 8 % C::ROW8 / 16, at, C::ROW8) * 16 + c16 % 2 * 8;
        *reinterpret_cast<uint2 *>(to) = hi;
        *reinterpret_cast<uint2 *>(to + TR_ROWS * D) = lo;
        if (C::F8 && c16 == 0) s.scale2[at] = a.c2 * __uint_as_float((254 - e) << 23);
      }
      async_fence();
      __syncwarp();
      if (lane == 0) bar_arrive(&s.q_ready);
    };
    auto load_queries = [&](const Walk &x) {
      if (C::F8 && x.tile < x.tiles - 1) load_split(x); else load_bf16(x);
    };
    bool live = w.next();
    if (live) load_queries(w);
    while (live) {
      const Walk cur = w;
      live = w.next();
      const int n = cur.count, h = cur.unit;
      const int len = length(cur.b);
      const bool has_nodes = cur.tile + n == cur.tiles;
      float cache_c2 = a.c2;
      if (C::F8 && cur.tile < cur.tiles - 1) {
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the split rows' scales are there ...
        if (on) cache_c2 = s.scale2[row];
        asm volatile("bar.sync 1, 256;" ::: "memory");  // ... and read, before the next segment's
      }
      int up = -2;  // the parent of node st, wanted at the segment's last tile
      if (has_nodes && st < a.n) up = a.parents[cur.b * a.ps[0] + st * a.ps[1]];
      uint64_t see = 0;  // the nodes that this row sees
      auto ancestors = [&] {
        // by pointer doubling: after k rounds a node knows 2^k of its line
        if (up < -1 || up >= st) up = -2;
        uint64_t mask = up == -2 ? 0 : 1ull << (st & 63);
        for (int step = 1;; step <<= 1) {
          if (st < TR_NODES) {
            s.anc[st] = mask;
            s.up[st] = (int8_t)up;
          }
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (step >= a.n) break;
          uint64_t over = 0;
          int next = -1;
          if (up >= 0) over = s.anc[up], next = s.up[up];
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (up >= 0) {
            mask = over ? mask | over : 0;  // a node below an unused one is unused
            up = over ? next : -2;
          }
        }
        if (on) see = s.anc[node];
      };
      float m = -INFINITY, l = 0.0f;  // the row's running maximum (log2 units), this thread's part of the sum
      for (int i = 0; i < n; ++i) {
        const uint32_t buf = (gt + i) & 1;
        const uint32_t at = lanes + C::COL_S + buf * KT;
        const bool nodes = cur.tile + i == cur.tiles - 1;
        if (nodes) ancestors();
        // (the length is first looked at where it matters: its load is long done by then)
        const int valid = nodes ? a.n : cur.tile + i < cur.tiles - 2 ? KT : min(KT, len - (cur.tile + i) * KT);
        const bool whole = valid == KT && !nodes;
        const int v64 = valid - 64 * half;
        const uint64_t keep = nodes ? (half ? 0 : see) : v64 >= 64 ? ~0ull : v64 > 0 ? (1ull << v64) - 1 : 0;
        const float c2 = nodes ? a.c2 : cache_c2;
        done(s.s_full, gt + i);
        // (FP8) the nodes' K is BF16: their scores need the queries as they are
        if (C::F8 && has_nodes && i == n - 2) load_bf16(cur);
        if (warp_on) {
          // S stays in registers between the maximum and the exponentials
          // where there are enough of them, and is read again where not (FP8)
          constexpr int HELD = C::F8 ? 32 : 64;
          uint32_t x[HELD];
          float top = -INFINITY;
          auto load = [&](int c) {
            uint32_t(&z)[32] = *reinterpret_cast<uint32_t(*)[32]>(x + (C::F8 ? 0 : 32 * c));
            tmem_ld32(z, at + 64 * half + 32 * c);
          };
          auto maximum = [&](int c) {
            const uint32_t *z = x + (C::F8 ? 0 : 32 * c), bits = (uint32_t)(keep >> (32 * c));
            if (whole) {
#pragma unroll
              for (int j = 0; j < 32; ++j) top = fmaxf(top, __uint_as_float(z[j]));
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) top = fmaxf(top, bits >> j & 1 ? __uint_as_float(z[j]) : -INFINITY);
            }
          };
          if (!C::F8) {
            load(0);
            load(1);
            tmem_wait_ld();
            maximum(0);
            maximum(1);
          } else {
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              load(c);
              tmem_wait_ld();
              maximum(c);
            }
          }
          s.share[exchange_slot(half, gt + i)][row] = top;
          asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
          top = fmaxf(top, s.share[exchange_slot(half ^ 1, gt + i)][row]) * c2;
          // the maximum moves only when it grows by more than 2^8: until then
          // weights up to 2^8 lose nothing in FP32 sums and BF16 products,
          // and the accumulator stays where it is
          const bool move = i == 0 || top > m + 8.0f;
          if (i > 0 && __any_sync(0xffffffffu, move)) {
            const float f = move ? exp2_fast(m - top) : 1.0f;
            done(s.o_done, gt + i - 1);
#pragma unroll 1
            for (int c = half * (D / 32); c < (half + 1) * (D / 32); ++c) {
              uint32_t o[16];
              tmem_ld16(o, lanes + 16 * c);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(lanes + 16 * c, o);
            }
            l *= f;
          }
          if (move) m = top;
          const float base2 = m == -INFINITY ? 0.0f : m;
          const uint64_t scale2 = pack2(c2, c2), minus2 = pack2(-base2, -base2);
          uint64_t sum = 0;  // two sums
#pragma unroll(C::F8 ? 1 : 2)
          for (int c = 0; c < 2; ++c) {
            if (C::F8) {
              load(c);
              tmem_wait_ld();
            }
            const uint32_t *z = x + (C::F8 ? 0 : 32 * c), bits = (uint32_t)(keep >> (32 * c));
            uint32_t y[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float p0, p1;
              unpack2(fma2(pack2(__uint_as_float(z[j]), __uint_as_float(z[j + 1])), scale2, minus2), p0, p1);
              p0 = exp2_fast(p0);
              p1 = exp2_fast(p1);
              if (!whole) {
                p0 = bits >> j & 1 ? p0 : 0.0f;
                p1 = bits >> (j + 1) & 1 ? p1 : 0.0f;
              }
              sum = add2(sum, pack2(p0, p1));
              y[j / 2] = pack_bf16(p0, p1);
            }
            // (over this thread's own, already read scores)
            tmem_st16(at + 64 * half + 16 * c, y);
          }
          float s0, s1;
          unpack2(sum, s0, s1);
          l += s0 + s1;
          tmem_wait_st();
          tc_fence_before();
        }
        if (!whole && (nodes || !C::F8)) {
          // V rows that no row may see are taken out of the product (0 * NaN is
          // NaN there): tokens behind the cache's length, unused nodes, and
          // values of a node that are not finite (its siblings do not see
          // them; the rows that do get them back below)
          // (the tile before is waited for so that a stage's parity names V(i)'s use of it)
          if (i > 0) done(s.o_done, gt + i - 1);
          const uint32_t v0 = base + (C::F8 ? i + (has_nodes ? 1 : 0) : pos_v(i, n)) * C::PIECES;
          const int from = nodes ? 0 : valid, to = nodes ? a.n : KT;
          for (int piece = from / C::VROWS; piece * C::VROWS < to; ++piece) {
            const uint32_t stage = (v0 + piece) % C::NSTAGE;
            wait(&s.full[stage], ((v0 + piece) / C::NSTAGE) & 1);
            uint8_t *v = ring + stage * C::STAGE;
            const int first = max(from - piece * C::VROWS, 0), last = min(to - piece * C::VROWS, C::VROWS);
            for (int x = first * (D / 8) + st; x < last * (D / 8); x += 256) {
              const int key = x / (D / 8), c16 = x % (D / 8);
              uint4 *p = reinterpret_cast<uint4 *>(v + (c16 / 8) * C::VROWS * 128 + key * 128 + (c16 % 8) * 16);
              if (!nodes || s.anc[piece * C::VROWS + key] == 0) {
                *p = make_uint4(0, 0, 0, 0);
                continue;
              }
              uint4 u = *p;
              uint32_t *e = reinterpret_cast<uint32_t *>(&u);
              bool found = false;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (not_finite_bf16(e[j])) e[j] &= 0xffff0000u, found = true;
                if (not_finite_bf16(e[j] >> 16)) e[j] &= 0x0000ffffu, found = true;
              }
              if (found) {
                *p = u;
                atomicOr(&s.bad, 1ull << (piece * C::VROWS + key));
              }
            }
          }
          async_fence();
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&s.p_ready[buf]);
      }
      // this segment's scores have all been read, so the tensor core is done
      // with its queries: the next segment's scores start beside the last product
      if (live) load_queries(w);
      // ---- the unit's rows, or this item's part of them
      const bool dead = has_nodes && see == 0;
      done(s.o_done, gt + n - 1);
      uint64_t bad = 0;
      if (has_nodes) {
        asm volatile("bar.sync 1, 256;" ::: "memory");
        bad = s.bad & see;
      }
      const bool direct = n == cur.tiles;
      if (warp_on) {
        // (the next write to either slot is behind the barrier that ends the segment)
        s.share[exchange_slot(half, gt + n)][row] = l;
        asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
        const int first = exchange_slot(0, gt + n);
        l = s.share[first][row] + s.share[first ^ 1][row];
        if (*abort) l = __uint_as_float(0x7fffffffu);
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const int64_t out_row = ((int64_t)cur.b * a.n + node) * (a.heads * a.group) + h * a.group + qg;
        const int64_t part_row = (int64_t)(2 * blockIdx.x + (walk.g < cur.start ? 1 : 0)) * a.rows + row;
#pragma unroll 1
        for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
          uint32_t x[32];
          tmem_ld32(x, lanes + 32 * c);
          tmem_wait_ld();
          if (bad)
            for (uint64_t rest = bad; rest; rest &= rest - 1) {
              const uint16_t *vn = a.vn + cur.b * a.vns[0] + h * a.vns[1] + (__ffsll((long long)rest) - 1) * a.vns[2] + 32 * c;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const uint32_t v = vn[j];
                if (not_finite_bf16(v)) x[j] = __float_as_uint(__uint_as_float(x[j]) + __uint_as_float(v << 16));
              }
            }
          if (!on) {
          } else if (direct) {
            uint32_t y[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              y[j] = dead ? 0u : pack_bf16(__uint_as_float(x[2 * j]) * inv, __uint_as_float(x[2 * j + 1]) * inv);
            uint4 *o = reinterpret_cast<uint4 *>(a.out + out_row * D + 32 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
          } else {
            uint4 *o = reinterpret_cast<uint4 *>(a.part + part_row * D + 32 * c);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
          }
          __syncwarp();
        }
        if (on && half == 0) {
          if (direct) a.lse[out_row] = dead ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
          else a.ml[part_row] = make_float2(m, dead ? -1.0f : l);
        }
        tc_fence_before();
      }
      // all have read O, s.bad and s.anc before the next segment's products and nodes
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (has_nodes && st == 0) s.bad = 0;
      base += (C::F8 ? n + (has_nodes ? 1 : 0) : 2 * n) * C::PIECES;
      gt += n;
    }
  } else if (C::F8 && (warp >= 12 || warp == 2 || warp == 3)) {
    // ---- FP8 caches: groups of TR_GROUP threads take the stages of V in turn,
    // turn their codes into BF16 and put them where TMA puts a BF16 stage.
    // The nodes' own K and V are BF16 and are copied.
    constexpr int GROUPS = 4, CHUNKS = C::RAW / 16 / TR_GROUP;  // 16-code pieces of one thread and stage
    constexpr uint32_t SLOTS = C::F8 ? C::NRAW : 1;
    const int ct = tid % TR_GROUP, grp = warp < 4 ? 0 : (warp - 10) / 2;
    static_assert(TR_GROUP == 64 && GROUPS % C::PIECES == 0, "groups of two warps, one stage each");
    static_assert(!C::F8 || (C::NRAW % GROUPS == 0 && C::NSTAGE % GROUPS == 0), "places of one group");
    // Piece j of this thread: key CHUNKS (ct / PER) + j of the stage's, dimensions 16 (ct % PER)...
    constexpr int PER = D / 16;
    static_assert(CHUNKS == 8, "a thread's keys cover a swizzle period");
    const int key = ct / PER * CHUNKS, unit = 2 * (ct % PER);  // unit: the first of its two 16-byte places in a row
    const int piece = grp % C::PIECES;
    Walk w = walk;
    uint32_t base = 0;  // tiles of the ring in the segments before
    bool ok = true;
    while (ok && w.next()) {
      const int n = w.count, len = length(w.b);
      const bool has_nodes = w.tile + n == w.tiles;
      const int tiles = n + (has_nodes ? 1 : 0), k_place = has_nodes ? nodes_k_place(n) : tiles;
      for (int t = (grp / C::PIECES - base % (GROUPS / C::PIECES) + GROUPS) % (GROUPS / C::PIECES); t < tiles;
           t += GROUPS / C::PIECES) {
        const bool is_k = t == k_place;
        const int i = is_k ? n - 1 : t - (t > k_place);  // the segment's tile
        const uint32_t seq = (base + t) * C::PIECES + piece, stage = seq % C::NSTAGE, slot = seq % SLOTS;
        uint8_t *to = ring + stage * C::STAGE;
        if (!(ok = wait(&s.raw_full[slot], (seq / SLOTS) & 1))) break;
        if (!(ok = wait(&s.empty[stage], ((seq / C::NSTAGE) & 1) ^ 1))) break;
        if (w.tile + i < w.tiles - 1) {
          const int left = len - (w.tile + i) * KT - piece * C::VROWS - key;  // keys from this thread's first
          const uint8_t *from = raw + slot * C::RAW + key * D + ct % PER * 16;
          uint8_t *at = to + (unit / 8) * C::VROWS * 128 + key * 128;
          uint32_t nan = 0;
          // (a short body: straight-line code for all pieces would wait for its instructions)
#pragma unroll 1
          for (int j = 0; j < CHUNKS; j += 2) {
            // (an odd key has its two units the other way round)
            uint8_t *y0 = at + j * 128 + ((unit & 7) ^ j) * 16, *y1 = at + j * 128 + ((unit & 7) ^ j ^ 1) * 16;
            const uint4 x0 = *reinterpret_cast<const uint4 *>(from + j * D);
            const uint4 x1 = *reinterpret_cast<const uint4 *>(from + j * D + D);
            uint4 lo, hi;
            e4m3_to_bf16(x0, lo, hi, nan);
            *reinterpret_cast<uint4 *>(y0) = lo;
            *reinterpret_cast<uint4 *>(y1) = hi;
            e4m3_to_bf16(x1, lo, hi, nan);
            *reinterpret_cast<uint4 *>(y1 + 128) = lo;
            *reinterpret_cast<uint4 *>(y0 + 128) = hi;
          }
          for (int j = max(left, 0); j < CHUNKS; ++j)  // behind the length
            for (int u = 0; u < 2; ++u) *reinterpret_cast<uint4 *>(at + j * 128 + (((unit & 7) ^ j) ^ u) * 16) = make_uint4(0, 0, 0, 0);
          if (nan & E4M3_NAN)
            for (int j = 0; j < CHUNKS; ++j)
              for (int u = 0; u < 2; ++u)
                e4m3_put_nan(reinterpret_cast<uint4 *>(at + j * 128 + (((unit & 7) ^ j) ^ u) * 16));
        } else {
          const uint16_t *src = is_k ? a.kn + w.b * a.kns[0] + w.unit * a.kns[1] : a.vn + w.b * a.vns[0] + w.unit * a.vns[1];
          const int64_t st = is_k ? a.kns[2] : a.vns[2];
          const int rows = is_k ? KT : C::VROWS, per = is_k ? 8 : D / 8;  // 16-byte units of a key in this stage
#pragma unroll 4
          for (int c = ct; c < C::STAGE / 16; c += TR_GROUP) {
            const int r = c / per, c16 = c % per;
            const int nd = is_k ? r : piece * C::VROWS + r, off = is_k ? piece * 8 + c16 : c16;
            const uint4 y = nd < a.n ? __ldg(reinterpret_cast<const uint4 *>(src + nd * st) + off) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(to + (c16 / 8) * rows * 128 + r * 128 + ((c16 ^ r) & 7) * 16) = y;
          }
        }
        async_fence();
        __syncwarp();
        if (lane == 0) {
          bar_arrive(&s.raw_empty[slot]);
          bar_arrive(&s.full[stage]);
        }
      }
      base += tiles;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// ---- joining the parts of a unit ---------------------------------------------

constexpr int TC_THREADS = 256, TC_MAX = 512;  // most items of a launch
constexpr int TC_BATCH = 8;                    // parts whose O a thread has in flight

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over the items c of a
// row's unit, in their order.  D / 4 threads hold a row's O.  With many items
// a unit a block has one row and its groups of threads share the parts; with
// few every group has a row of its own.  What bounds it is latency: the parts
// are in L2, and all loads of a thread are issued before the first is used.
template <int D, bool FEW>
__global__ void __launch_bounds__(TC_THREADS) k_tree_combine(const __grid_constant__ TreeArgs a, int groups) {
  constexpr int LANES = D / 4, GROUPS = TC_THREADS / LANES;
  __shared__ int32_t s_pre[PLAN_BATCH + 1];
  __shared__ float2 s_ml[FEW ? 1 : TC_MAX];
  __shared__ float s_red[1][TC_THREADS / 32];
  __shared__ float4 s_o[FEW ? 1 : GROUPS][LANES];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = tid / LANES, d4 = tid % LANES;
  grid_dependency_release();
  // (the lengths are older than the attention kernel, which released this one
  // after its own wait)
  if (warp == 0) tile_prefix<TR_KEYS>(a.lengths, a.len_stride, a.t, a.batch, 1 + TR_IDLE, nullptr, s_pre);
  __syncthreads();
  const int rows = a.n * a.group, all = rows * a.heads * a.batch;
  const int index = FEW ? blockIdx.x * GROUPS + group : blockIdx.x;
  if (index >= all) return;  // (of the last block, where FEW: no barrier of the block below)
  const int r = index % rows, bh = index / rows, h = bh % a.heads, b = bh / a.heads;
  const int mt = r / TR_ROWS, places = s_pre[b + 1] - s_pre[b];
  const Plan plan((long long)s_pre[a.batch] * a.heads, groups);
  const long long g0 = (long long)s_pre[b] * a.heads + (long long)h * places;
  const int c0 = plan.owner(g0), c1 = plan.owner(g0 + places - TR_IDLE - 1);
  const int shift = plan.begin(c0) < g0 ? 1 : 0;  // only its first item may hold a part of a unit before
  // (blocks without work wait too: what follows this kernel on the stream
  // must find the attention kernel's own rows written)
  grid_dependency_wait();
  if (c0 == c1) return;  // written by its one CTA
  const int parts = c1 - c0 + 1, prow = r - mt * TR_ROWS;
  auto slot = [&](int i) { return (int64_t)(2 * ((c0 + i) * a.mtiles + mt) + (i == 0 ? shift : 0)) * a.rows + prow; };
  auto o_of = [&](int i) { return __ldcg(reinterpret_cast<const float4 *>(a.part + slot(i) * D) + d4); };
  const int first = FEW ? 0 : group, gap = FEW ? 1 : GROUPS;
  float4 x[TC_BATCH];
#pragma unroll
  for (int k = 0; k < TC_BATCH; ++k)
    if (first + k * gap < parts) x[k] = o_of(first + k * gap);
  // the row's maximum, its sum, and whether it is unused (l < 0 in a part)
  float m = -INFINITY, l = 0.0f;
  bool dead = false;
  if (FEW) {
    for (int i = 0; i < parts; ++i) m = fmaxf(m, __ldcg(a.ml + slot(i)).x);
  } else {
    for (int i = tid; i < parts; i += TC_THREADS) {
      s_ml[i] = __ldcg(a.ml + slot(i));
      m = fmaxf(m, s_ml[i].x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_red[0][warp] = m;
    __syncthreads();
    m = s_red[0][0];
#pragma unroll
    for (int i = 1; i < TC_THREADS / 32; ++i) m = fmaxf(m, s_red[0][i]);
  }
  const float base = m == -INFINITY ? 0.0f : m;
  float4 o = make_float4(0, 0, 0, 0);
  auto ml_of = [&](int i) { return FEW ? __ldcg(a.ml + slot(i)) : s_ml[i]; };
  auto add = [&](const float4 &v, int i) {
    const float2 ml = ml_of(i);
    const float w = exp2_fast(ml.x - base);
    dead = dead || ml.y < 0.0f;
    l += w * ml.y;
    // (also where w is 0: a value that is not finite counts however small its
    // weight is, as it does inside a part; an unused row's sums are not used)
    o.x = fmaf(w, v.x, o.x);
    o.y = fmaf(w, v.y, o.y);
    o.z = fmaf(w, v.z, o.z);
    o.w = fmaf(w, v.w, o.w);
  };
#pragma unroll
  for (int k = 0; k < TC_BATCH; ++k)
    if (first + k * gap < parts) add(x[k], first + k * gap);
  for (int i = first + TC_BATCH * gap; i < parts; i += gap) add(o_of(i), i);
  if (!FEW) {
    // the groups' parts, in order
    s_o[group][d4] = o;
    __syncthreads();
    float *sums = reinterpret_cast<float *>(s_pre);  // (its last use is above)
    if (d4 == 0) sums[group] = dead ? -INFINITY : l;
    __syncthreads();
    if (group) return;
    l = 0.0f;
    dead = false;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      dead = dead || sums[i] == -INFINITY;
      l += sums[i];
      if (i) {
        const float4 v = s_o[i][d4];
        o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
      }
    }
  }
  const int node = r / a.group;
  const int64_t row = ((int64_t)b * a.n + node) * (a.heads * a.group) + h * a.group + (r - node * a.group);
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const uint2 y = dead ? make_uint2(0, 0) : make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  reinterpret_cast<uint2 *>(a.out + row * D)[d4] = y;
  if (d4 == 0) a.lse[row] = dead ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <class C>
int launch_tree(const TreeMaps &maps, const TreeArgs &a, int ctas, int device, cudaStream_t st) {
  constexpr int smem = C::RING + (int)sizeof(TreeSmem<C>);
  static_assert(smem <= 232448, "shared memory");
  auto *kernel = &k_tree_attention<C>;
  static bool set[64];
  if (int rc = op_shared_memory(reinterpret_cast<const void *>(kernel), smem, device, set)) return rc;
  if (int rc = op_cuda(op_launch(kernel, dim3(ctas), dim3(C::THREADS), smem, st, 1, maps, a),
                       "k_tree_attention launch"))
    return rc;
  if (a.whole) return SKV_OK;
  const unsigned rows = (unsigned)(a.batch * a.heads * a.n * a.group);
  const int items = ctas / a.mtiles;
  constexpr unsigned per = TC_THREADS / (C::D / 4);
  // (a unit has about items / units parts: more than one thread group's batch of them is shared)
  const bool few = items <= (TC_BATCH - 2) * a.batch * a.heads;
  return op_cuda(few ? op_launch(k_tree_combine<C::D, true>, dim3((rows + per - 1) / per), dim3(TC_THREADS), 0, st, 1, a, items)
                     : op_launch(k_tree_combine<C::D, false>, dim3(rows), dim3(TC_THREADS), 0, st, 1, a, items),
                 "k_tree_combine launch");
}

template <bool F8>
int launch_tree_d(int d, const TreeMaps &maps, const TreeArgs &a, int ctas, int device, cudaStream_t st) {
  if (d == 64) return launch_tree<TreeCfg<64, F8>>(maps, a, ctas, device, st);
  if (d == 128) return launch_tree<TreeCfg<128, F8>>(maps, a, ctas, device, st);
  return launch_tree<TreeCfg<256, F8>>(maps, a, ctas, device, st);
}

// Whether units are left whole: one CTA each, one launch and no workspace.
// Cutting them shares their tiles among all SMs, tiles (1 - units / sms) less
// for the longest, and costs the partials and a second kernel.  Measured (BF16,
// a tile 1.2 us): 12 units, 128 tokens 8.7 us whole, 10.4 cut; 512, 12.3 and
// 11.0 (and 4 us less on the host); 1152, 17.9 and 10.9.  128 units, 128
// tokens 9.6 and 15.2; 2176, 30.7 and 35.9.
bool tree_whole(int sms, int64_t batch, int64_t heads, int64_t mtiles, int64_t t) {
  const int64_t units = batch * heads * mtiles, tiles = (t + TR_KEYS - 1) / TR_KEYS + 1;
  return units <= sms && tiles * (sms - units) <= TR_JOIN * sms;
}

// CTAs of a launch: one per SM, whole items (or fewer, the most places that the list can have).
int64_t tree_ctas(int sms, int64_t batch, int64_t heads, int64_t mtiles, int64_t t) {
  const int64_t most = batch * heads * ((t + TR_KEYS - 1) / TR_KEYS + 1 + TR_IDLE);
  const int64_t c = sms > mtiles ? (sms / mtiles < TC_MAX ? sms / mtiles : TC_MAX) : 1;
  return (most < c ? most : c) * mtiles;
}

int64_t tree_workspace(int sms, const SkvTree *d) {
  const int64_t rows = d->n * (d->heads / d->kv_heads), per = rows < TR_ROWS ? rows : TR_ROWS;
  const int64_t mtiles = (rows + TR_ROWS - 1) / TR_ROWS;
  auto slots = [&](int64_t batch) {  // of a launch
    return batch == 0 || tree_whole(sms, batch, d->kv_heads, mtiles, d->tokens)
               ? 0
               : 2 * tree_ctas(sms, batch, d->kv_heads, mtiles, d->tokens);
  };
  const int64_t full = slots(d->batch < PLAN_BATCH ? d->batch : PLAN_BATCH), last = slots(d->batch % PLAN_BATCH);
  return (full > last ? full : last) * per * (d->dim + 2) * 4;
}

int check_tree(const SkvTree *d) {
  if (!d) return op_fail(SKV_E_INVALID, "null descriptor");
  if (d->dim != 64 && d->dim != 128 && d->dim != 256) return op_fail(SKV_E_INVALID, "head size must be 64, 128 or 256");
  if (d->n < 1 || d->n > TR_NODES) return op_fail(SKV_E_INVALID, "nodes must be in [1, %d]", TR_NODES);
  if (d->kv_heads < 1 || d->heads < 1 || d->heads % d->kv_heads || d->heads > 4096)
    return op_fail(SKV_E_INVALID, "query heads must be a multiple of the KV heads, and at most 4096");
  if (d->batch < 0 || d->batch > INT32_MAX / (d->heads * d->n))
    return op_fail(SKV_E_INVALID, "batch * nodes * query heads must be below 2^31");
  if (d->tokens < 1 || d->tokens > (1 << 26)) return op_fail(SKV_E_INVALID, "tokens must be in [1, 2^26]");
  if (!(d->scale > 0.0) || !(d->scale < 1e30)) return op_fail(SKV_E_INVALID, "scale must be positive and finite");
  if (d->cache_dtype != SKV_DTYPE_BF16 && d->cache_dtype != SKV_DTYPE_E4M3)
    return op_fail(SKV_E_INVALID, "the cache is BF16 or FP8 e4m3");
  return SKV_OK;
}

}  // namespace

int record_maps(CUtensorMap *two, const uint8_t *records, int64_t rows) {
  const int64_t step[3] = {REC, 0, 0};
  for (int i = 0; i < 2; ++i)
    if (int rc = make_byte_map(two + i, records + i * D, D, rows, 1, 1, step, i ? TR_KEYS / (D / 64) : TR_KEYS, i ? D : 128, !i))
      return rc;
  return SKV_OK;
}

int tree_attention(const SkvTree *d, const CUtensorMap *cells, const int32_t *tlen, uint32_t *status, cudaStream_t st) {
  if (int rc = check_tree(d)) return rc;
  if (d->batch == 0) return SKV_OK;
  if (!d->q || !d->k || !d->v || !d->parents || !d->out || !d->lse ||
      (!cells && (!d->k_cache || !d->v_cache || !d->lengths)))
    return op_fail(SKV_E_INVALID, "null input or output pointer");
  const bool f8 = d->cache_dtype == SKV_DTYPE_E4M3;
  const int64_t of_q[3] = {d->batch, d->n, d->heads}, of_cache[3] = {d->batch, d->kv_heads, d->tokens},
                of_nodes[3] = {d->batch, d->kv_heads, d->n};
  struct Rows {
    const void *base;
    const int64_t *given, *size;
    int64_t unit, stride[3];
  } rows_of[5] = {{d->q, d->q_stride, of_q, 8, {}},
                  {d->k, d->k_stride, of_nodes, 8, {}},
                  {d->v, d->v_stride, of_nodes, 8, {}},
                  {d->k_cache, d->k_cache_stride, of_cache, f8 ? 16 : 8, {}},
                  {d->v_cache, d->v_cache_stride, of_cache, f8 ? 16 : 8, {}}};
  for (int i = 0; i < (cells ? 3 : 5); ++i) {
    Rows &x = rows_of[i];
    op_strides(x.stride, x.given, x.size, 3);
    if (x.given[3] != 1) return op_fail(SKV_E_INVALID, "the innermost dimension must be contiguous");
    bool ok = (uintptr_t)x.base % 16 == 0;
    for (int j = 0; j < 3; ++j) ok = ok && x.stride[j] >= 0 && x.stride[j] % x.unit == 0;
    if (!ok) return op_fail(SKV_E_INVALID, "rows must start on 16-byte boundaries");
    if (i && x.size[2] > 1 && x.stride[2] == 0) return op_fail(SKV_E_INVALID, "tokens must not share one row");
  }
  if ((uintptr_t)d->out % 16 || (uintptr_t)d->workspace % 16)
    return op_fail(SKV_E_INVALID, "outputs must start on 16-byte boundaries");
  const int64_t *const qs = rows_of[0].stride, *const ks = rows_of[1].stride, *const vs = rows_of[2].stride,
                *const kcs = rows_of[3].stride, *const vcs = rows_of[4].stride;
  int sms = 0;
  if (int rc = sm_count(d->device, &sms)) return rc;
  DeviceScope scope((int)d->device);
  if (int rc = op_cuda(scope.error(), "selecting the device")) return rc;
  const int64_t scratch = tree_workspace(sms, d);
  if (d->workspace_bytes < scratch || (scratch && !d->workspace))
    return op_fail(SKV_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)d->workspace_bytes, (long long)scratch);
  TreeArgs a{};
  a.status = status;
  if (!status)
    if (int rc = status_word((int)d->device, &a.status)) return rc;
  const int group = (int)(d->heads / d->kv_heads), rows = (int)d->n * group;
  a.heads = (int)d->kv_heads, a.group = group, a.n = (int)d->n, a.t = (int)d->tokens;
  a.by_group = ((1ull << 32) + group - 1) / group;
  a.mtiles = (rows + TR_ROWS - 1) / TR_ROWS;
  a.rows = rows < TR_ROWS ? rows : TR_ROWS;
  a.c2 = (float)(d->scale * 1.4426950408889634);
  a.len_stride = cells || d->batch == 1 ? 0 : d->lengths_stride;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = qs[i];
    a.kns[i] = ks[i], a.vns[i] = vs[i];
  }
  op_strides(a.ps, d->parents_stride, of_q, 2);
  for (int64_t b0 = 0; b0 < d->batch; b0 += PLAN_BATCH) {
    const int64_t nb = d->batch - b0 < PLAN_BATCH ? d->batch - b0 : PLAN_BATCH;
    a.batch = (int)nb;
    a.q = static_cast<const uint16_t *>(d->q) + b0 * a.qs[0];
    a.kn = static_cast<const uint16_t *>(d->k) + b0 * a.kns[0];
    a.vn = static_cast<const uint16_t *>(d->v) + b0 * a.vns[0];
    a.cell_maps = cells ? cells + 2 * b0 * d->kv_heads : nullptr;
    a.lengths = cells ? tlen : static_cast<const int32_t *>(d->lengths) + b0 * a.len_stride;
    a.parents = static_cast<const int32_t *>(d->parents) + b0 * a.ps[0];
    a.out = static_cast<uint16_t *>(d->out) + b0 * d->n * d->heads * d->dim;
    a.lse = static_cast<float *>(d->lse) + b0 * d->n * d->heads;
    a.whole = tree_whole(sms, nb, a.heads, a.mtiles, d->tokens);
    const int ctas = a.whole ? (int)(nb * a.heads * a.mtiles) : (int)tree_ctas(sms, nb, a.heads, a.mtiles, d->tokens);
    a.part = static_cast<float *>(d->workspace);
    a.ml = reinterpret_cast<float2 *>(a.part + 2 * (int64_t)ctas * a.rows * d->dim);
    TreeMaps maps{};
    int rc = SKV_OK;
    if (!f8) {
      const int pieces = (int)d->dim / 64;
      const struct {
        CUtensorMap *map;
        const void *base;
        const int64_t *s;
        int64_t rows;
      } four[4] = {{&maps.k, static_cast<const uint16_t *>(d->k_cache) + b0 * kcs[0], kcs, d->tokens},
                   {&maps.v, static_cast<const uint16_t *>(d->v_cache) + b0 * vcs[0], vcs, d->tokens},
                   {&maps.kn, a.kn, ks, d->n},
                   {&maps.vn, a.vn, vs, d->n}};
      for (int i = 0; i < 4 && !rc; ++i) {
        const int64_t step[3] = {four[i].s[2], four[i].s[1], four[i].s[0]};
        rc = make_map(four[i].map, four[i].base, d->dim, four[i].rows, d->kv_heads, nb, step,
                      i % 2 ? TR_KEYS / pieces : TR_KEYS, i % 2 ? pieces : 1);  // K: one piece, V: all of a row
        a.along[i][0] = d->kv_heads > 1 && four[i].s[1] ? 1 : 0;
        a.along[i][1] = nb > 1 && four[i].s[0] ? 1 : 0;
      }
    } else if (!cells) {
      for (int i = 0; i < 2 && !rc; ++i) {
        const int64_t *at = i ? vcs : kcs, step[3] = {at[2], at[1], at[0]};
        const void *base = static_cast<const uint8_t *>(i ? d->v_cache : d->k_cache) + b0 * at[0];
        rc = make_byte_map(i ? &maps.v : &maps.k, base, d->dim, d->tokens, d->kv_heads, nb, step,
                           i ? TR_KEYS / ((int)d->dim / 64) : TR_KEYS, i ? (int)d->dim : d->dim == 64 ? 64 : 128, !i);
        a.along[i][0] = d->kv_heads > 1 && at[1] ? 1 : 0;
        a.along[i][1] = nb > 1 && at[0] ? 1 : 0;
      }
    }
    if (!rc) rc = f8 ? launch_tree_d<true>((int)d->dim, maps, a, ctas, (int)d->device, st) : launch_tree_d<false>((int)d->dim, maps, a, ctas, (int)d->device, st);
    if (rc) return rc;
  }
  return SKV_OK;
}

}  // namespace skv

extern "C" {

int skv_tree_attention(const SkvTree *d, void *stream) {
  return skv::tree_attention(d, nullptr, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

int skv_tree_workspace(const SkvTree *d, int64_t *bytes) {
  using namespace skv;
  if (!bytes) return op_fail(SKV_E_INVALID, "null result pointer");
  if (int rc = check_tree(d)) return rc;
  int sms = 0;
  if (int rc = sm_count(d->device, &sms)) return rc;
  *bytes = tree_workspace(sms, d);
  return SKV_OK;
}

int skv_operator_status(int32_t device, uint32_t *flags) {
  using namespace skv;
  if (!flags) return op_fail(SKV_E_INVALID, "null result pointer");
  DeviceScope scope(device);
  if (int rc = op_cuda(scope.error(), "selecting the device")) return rc;
  uint32_t *word = nullptr, got = 0;
  if (int rc = status_word(device, &word)) return rc;
  if (int rc = op_cuda(cudaDeviceSynchronize(), "waiting for the device")) return rc;
  if (int rc = op_cuda(cudaMemcpy(&got, word, sizeof got, cudaMemcpyDeviceToHost), "reading the status word")) return rc;
  if (got)  // reported once: later calls are judged by themselves
    if (int rc = op_cuda(cudaMemset(word, 0, sizeof got), "clearing the status word")) return rc;
  *flags = got;
  return SKV_OK;
}

}  // extern "C"
