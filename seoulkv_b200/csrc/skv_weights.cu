// skv_weights.cu -- attention weights accumulated per cached key.
//
//   out[t] = w[t] + sum over the rows r of a KV head of exp(scale q_r.k_t - lse_r)
//
// for t below the sequence's length; elsewhere out[t] = w[t].  With the rows'
// log-sum-exp known, a key's sum needs no other key: one pass over K.
//
// The product runs on tcgen05 with the keys as M = 128 lanes and the rows as
// N: every thread of the epilogue then holds one key's scores in its own lane
// and sums their exponentials without a word to its neighbours, in a fixed
// order.  A tile's K arrives as pieces of 128 keys x 128 bytes (16 KB), so
// that the ring stays deep beside up to 128 KB of queries in shared memory;
// the accumulator (FP32, tensor memory) is double-buffered against two
// epilogue groups.  CTAs take contiguous ranges of the list of all tiles.
//
// An FP8 cache goes to the tensor core as it is stored: the queries are split
// into two FP8 rows whose sum they are (skv_tensor.cuh), with a power of two
// per row that the epilogue takes out again.
//
// What bounds it, measured at 16 query heads on 4 KV heads of 256 (a copy
// moves 6437 GB/s): one token over 131072 cached, 44.1 us, 273 MB = 96%; the
// last 32 tokens (128 rows) of four requests of up to 32768, 31.7 us, 139 MB =
// 68%.  Longer caches add bytes at 6.7 TB/s, so what is left is a fixed 8 us:
// lengths, queries and the first tile come one after the other, the last
// epilogue follows the last tile, and a CTA whose range passes from one head to
// the next reloads its queries while its ring stands full.  Over FP8: one token
// over 131072, 28.4 us, 138 MB = 76% (262144: 48.4 us, 89%).
#include <cuda_bf16.h>

#include "skv_ops.cuh"
#include "skv_plan.cuh"
#include "skv_tensor.cuh"

namespace skv {
namespace {

constexpr int WT_KEYS = 128, WT_PIECE = WT_KEYS * 128;  // bytes of a piece
constexpr int WT_ROWS = 256;                            // rows of one launch: the MMA's largest N
constexpr int WT_STAGES = 12;
constexpr int WT_THREADS = 384;

struct WeightsArgs {
  const uint16_t *q;
  int64_t qs[3];  // element strides (sequence, node, head)
  const int32_t *lengths;
  int64_t len_stride;
  const float *lse;
  int64_t ls[3];  // (sequence, node, head)
  const uint8_t *take;  // [sequence][node]: rows that count (null: all)
  int64_t ts[2];
  const float *w;
  float *out;
  int64_t ws[3], os[3];  // (sequence, head, token)
  uint64_t by_group;  // (by_inverse)
  int32_t batch, heads, group, t, row0, rows, cols;  // rows [row0, row0 + rows) of a head, counted from q's node; cols: rows up to 16s
  int32_t along[2];
  int32_t stages;  // pieces of the ring
  float scale;
  uint32_t *status;
};

struct WeightsSmem {
  uint64_t full[WT_STAGES], empty[WT_STAGES];
  uint64_t q_ready, q_free, acc_full[2], acc_free[2], drain;
  uint32_t tmem, abort;
  alignas(16) float lse[2][WT_ROWS];  // +inf for rows that do not count
  alignas(16) float scale[2][WT_ROWS];  // over an FP8 cache: the scale, by the row's power of two
  int64_t q_at[WT_ROWS];               // element offsets of the rows in a head's queries
  int32_t len[PLAN_BATCH];
  int32_t pre[PLAN_BATCH + 1];
};

template <int D, bool F8>
__global__ void __launch_bounds__(WT_THREADS, 1)
    k_weights(const __grid_constant__ CUtensorMap map, const __grid_constant__ WeightsArgs a) {
  // bytes of a piece's rows, pieces of a tile; FP8 queries: hi's pieces, then lo's
  constexpr int ROW = F8 && D == 64 ? 64 : 128, SUB = D * (F8 ? 1 : 2) / ROW, PIECE = WT_KEYS * ROW;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t *queries = smem_dyn + (1024 - (s_addr(smem_dyn) & 1023)) % 1024;  // [piece][cols][ROW bytes], swizzled
  uint8_t *ring = queries + a.cols * D * 2;
  WeightsSmem &s = *reinterpret_cast<WeightsSmem *>(ring + a.stages * WT_PIECE);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int stages = a.stages;
  if (warp == 0) {
    if (lane == 0) tma_prefetch_map(&map);
    grid_dependency_wait();
    tile_prefix<WT_KEYS>(a.lengths, a.len_stride, a.t, a.batch, 0, s.len, s.pre);
  } else if (warp == 1) {
    tmem_alloc(&s.tmem, 512);
  } else if (warp == 2 && lane == 0) {
    for (int i = 0; i < stages; ++i) {
      bar_init(&s.full[i], 1);
      bar_init(&s.empty[i], 1);
    }
    bar_init(&s.q_ready, 8);
    bar_init(&s.q_free, 1);
    bar_init(&s.drain, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(&s.acc_full[i], 1);
      bar_init(&s.acc_free[i], 4);
    }
    bar_init_fence();
    s.abort = 0;
  }
  grid_dependency_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_release();
  const uint32_t tmem = *(volatile uint32_t *)&s.tmem;
  volatile uint32_t *abort = &s.abort;
  const long long total = (long long)s.pre[a.batch] * a.heads;
  const Plan plan(total, (int)gridDim.x);
  const int cta = blockIdx.x;
  const long long g_begin = plan.begin(cta), g_end = plan.begin(cta + 1);
  auto wait = [&](uint64_t *bar, uint32_t parity) { return bar_wait(bar, parity, abort, a.status); };

  if (warp == 0) {
    // ---- loads
    const uint32_t one = elect_lane();
    Walk w(s.pre, a.batch, a.heads, 0, g_begin, g_end);
    uint32_t seq = 0;
    int stage = 0;
    uint32_t turn = 0;
    bool ok = true;
    while (ok && w.next())
      for (int i = 0; i < w.count && ok; ++i)
        for (int sub = 0; sub < SUB; ++sub) {
          if (!(ok = wait(&s.empty[stage], turn ^ 1))) break;
          const int row = (w.tile + i) * WT_KEYS, y = w.unit * a.along[0], z = w.b * a.along[1];
          uint8_t *to = ring + stage * WT_PIECE;
          if (F8)
            tma_load_bytes(one, to, &map, sub * ROW, row, y, z, &s.full[stage], PIECE);
          else
            tma_load(one, to, &map, row, sub, y, z, &s.full[stage], PIECE);
          ++seq;
          if (++stage == stages) stage = 0, turn ^= 1;
        }
    if (!ok)  // gave up: the copies in flight still land before the CTA ends
      for (uint32_t back = 1; back <= (uint32_t)stages && back <= seq; ++back) {
        const uint32_t q = seq - back;
        const unsigned long long t0 = timer_ns();
        while (!bar_try(&s.full[q % stages], (q / stages) & 1) && timer_ns() - t0 < WAIT_NS / 4) {
        }
      }
  } else if (warp == 1) {
    // ---- tensor core
    const uint32_t one = elect_lane();
    Walk w(s.pre, a.batch, a.heads, 0, g_begin, g_end);
    const uint32_t desc = F8 ? mma_desc_f8(WT_KEYS, a.cols) : mma_desc(WT_KEYS, a.cols, false);
    const uint32_t q0 = s_addr(queries), ring0 = s_addr(ring);
    int stage = 0;
    uint32_t turn = 0, gt = 0, seg = 0;
    while (w.next()) {
      wait(&s.q_ready, seg & 1);
      for (int i = 0; i < w.count; ++i, ++gt) {
        const uint32_t buf = gt & 1;
        wait(&s.acc_free[buf], ((gt >> 1) & 1) ^ 1);
        tc_fence_after();
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
          wait(&s.full[stage], turn);
          const uint32_t k0 = ring0 + stage * WT_PIECE, qs = q0 + sub * a.cols * ROW, d = tmem + buf * WT_ROWS;
#pragma unroll
          for (int ks = 0; ks < ROW / 32; ++ks) {
            const uint64_t kd = smem_desc_rows(k0 + ks * 32, ROW), qd = smem_desc_rows(qs + ks * 32, ROW);
            if (F8) {
              mma_f8(one, d, kd, qd, desc, sub + ks > 0);
              mma_f8(one, d, kd, smem_desc_rows(qs + a.cols * D + ks * 32, ROW), desc, true);
            } else {
              mma_ss(one, d, kd, qd, desc, sub + ks > 0);
            }
          }
          mma_commit(one, &s.empty[stage]);
          if (++stage == stages) stage = 0, turn ^= 1;
        }
        mma_commit(one, &s.acc_full[buf]);
      }
      mma_commit(one, &s.q_free);
      ++seg;
    }
    if (*abort) {  // what was issued ends before tensor memory is given back
      mma_commit(one, &s.drain);
      const unsigned long long t0 = timer_ns();
      while (!bar_try(&s.drain, 0) && timer_ns() - t0 < WAIT_NS / 4) {
      }
    }
  } else if (warp < 4) {
    // ---- tokens behind the lengths keep their weights
    if (a.w != a.out) {
      const int pairs = a.batch * a.heads, ctas = (int)gridDim.x;
      const int share = ctas > pairs ? ctas / pairs : 1;  // CTAs of one (sequence, head)
      for (int p = cta / share; p < pairs; p += (ctas + share - 1) / share) {
        const int b = p / a.heads, h = p - b * a.heads;
        const float *w = a.w + b * a.ws[0] + h * a.ws[1];
        float *o = a.out + b * a.os[0] + h * a.os[1];
        constexpr int BATCH = 8;  // (loads in flight: one at a time this copy outlasted the rest of the kernel)
        for (int t0 = s.len[b] + (cta % share) * 64 + tid - 64; t0 < a.t; t0 += share * 64 * BATCH) {
          float x[BATCH];
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            const int t = t0 + share * 64 * j;
            x[j] = t < a.t ? w[t * a.ws[2]] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            const int t = t0 + share * 64 * j;
            if (t < a.t) o[t * a.os[2]] = x[j];
          }
        }
      }
    }
  } else if (warp < 12) {
    // ---- epilogue: one key per thread, tiles in turn between the two groups
    const int et = tid - 128, half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp - 4) & 3) << 21) + half * WT_ROWS;
    Walk w(s.pre, a.batch, a.heads, 0, g_begin, g_end);
    uint32_t gt = 0, seg = 0;
    while (w.next()) {
      const int h = w.unit;
      // the head's rows, once the tensor core is done with the ones before
      if (seg) wait(&s.q_free, (seg - 1) & 1);
      if (et < a.cols) {
        const int row = a.row0 + min(et, a.rows - 1), node = by_inverse(row, a.by_group), g = row - node * a.group;
        const float l = a.lse[w.b * a.ls[0] + node * a.ls[1] + (h * a.group + g) * a.ls[2]];
        const uint8_t take = a.take ? a.take[w.b * a.ts[0] + node * a.ts[1]] : 1;
        // (-inf: a row that saw nothing)
        s.lse[seg & 1][et] = et < a.rows && take && l != -INFINITY ? l : INFINITY;
        s.q_at[et] = node * a.qs[1] + g * a.qs[2];
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
      const int c16 = et % (D / 8);
      const uint16_t *q = a.q + w.b * a.qs[0] + h * a.group * a.qs[2] + c16 * 8;
      // (short loops: code that runs once per launch waits for its
      // instructions, and unrolled loads took 20000 cycles here)
      if (F8) {
        uint4 v = make_uint4(0, 0, 0, 0), ahead = v;
        auto fetch = [&](int r) { return r < a.cols && s.lse[seg & 1][r] != INFINITY ? __ldg(reinterpret_cast<const uint4 *>(q + s.q_at[r])) : make_uint4(0, 0, 0, 0); };
        ahead = fetch(et / (D / 8));
#pragma unroll 1
        for (int r = et / (D / 8); r < a.cols; r += 256 / (D / 8)) {
          v = ahead;
          ahead = fetch(r + 256 / (D / 8));
          const uint32_t e = split_exponent(v, D / 8);
          uint2 hi, lo;
          split_eight(v, __uint_as_float(e << 23), hi, lo);
          // 8 bytes at byte 8 c16 of the row
          uint8_t *to = queries + (c16 * 8 / ROW) * a.cols * ROW + r * ROW + swizzled(c16 * 8 % ROW / 16, r, ROW) * 16 + c16 % 2 * 8;
          *reinterpret_cast<uint2 *>(to) = hi;
          *reinterpret_cast<uint2 *>(to + a.cols * D) = lo;
          if (c16 == 0) s.scale[seg & 1][r] = a.scale * __uint_as_float((254 - e) << 23);
        }
      } else {
        uint8_t *to = queries + (c16 / 8) * a.cols * 128;
#pragma unroll 1
        for (int r = et / (D / 8); r < a.cols; r += 256 / (D / 8))
          cp_async16(to + r * 128 + ((c16 % 8) ^ (r & 7)) * 16, q + s.q_at[r], s.lse[seg & 1][r] != INFINITY);
        cp_async_wait();
      }
      async_fence();
      __syncwarp();
      if (lane == 0) bar_arrive(&s.q_ready);
      if (F8) asm volatile("bar.sync 2, 256;" ::: "memory");  // the rows' scales are there
      const float4 *scale = reinterpret_cast<const float4 *>(s.scale[seg & 1]);
      const float4 *lse = reinterpret_cast<const float4 *>(s.lse[seg & 1]);
      const float *wrow = a.w + w.b * a.ws[0] + h * a.ws[1];
      float *orow = a.out + w.b * a.os[0] + h * a.os[1];
      for (int i = 0; i < w.count; ++i, ++gt) {
        if ((gt & 1) != (uint32_t)half) continue;
        const int t = (w.tile + i) * WT_KEYS + (et & 127);
        const bool on = t < s.len[w.b];
        const float before = on ? wrow[t * a.ws[2]] : 0.0f;
        wait(&s.acc_full[half], (gt >> 1) & 1);
        __syncwarp();
        tc_fence_after();
        float sum[4] = {0, 0, 0, 0};
        for (int c = 0; c < a.cols; c += 16) {
          uint32_t x[16];
          tmem_ld16(x, lanes + c);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // (the difference first: rounded in log2 units, score and lse
            // would each bring their own size's error into the exponent)
            const float4 l = lse[c / 4 + j], f = F8 ? scale[c / 4 + j] : make_float4(a.scale, a.scale, a.scale, a.scale);
            sum[0] += exp2_fast(fmaf(__uint_as_float(x[4 * j]), f.x, -l.x) * 1.4426950408889634f);
            sum[1] += exp2_fast(fmaf(__uint_as_float(x[4 * j + 1]), f.y, -l.y) * 1.4426950408889634f);
            sum[2] += exp2_fast(fmaf(__uint_as_float(x[4 * j + 2]), f.z, -l.z) * 1.4426950408889634f);
            sum[3] += exp2_fast(fmaf(__uint_as_float(x[4 * j + 3]), f.w, -l.w) * 1.4426950408889634f);
          }
        }
        float add = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        // a key with an infinity or a NaN: the zeros that stand for rows that
        // do not count made NaNs with it, so they are left out one by one
        if (__any_sync(0xffffffffu, add != add)) {
          float again = 0.0f;
#pragma unroll 1
          for (int c = 0; c < a.cols; c += 16) {
            uint32_t x[16];
            tmem_ld16(x, lanes + c);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float l = s.lse[seg & 1][c + j], f = F8 ? s.scale[seg & 1][c + j] : a.scale;
              if (l != INFINITY) again += exp2_fast(fmaf(__uint_as_float(x[j]), f, -l) * 1.4426950408889634f);
            }
          }
          if (add != add) add = again;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&s.acc_free[half]);
        if (*abort) add = __uint_as_float(0x7fffffffu);
        if (on) orow[t * a.os[2]] = before + add;
      }
      ++seg;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

template <int D, bool F8>
int launch_weights(const CUtensorMap &map, WeightsArgs &a, int sms, int device, cudaStream_t st) {
  constexpr int most = 232448, fixed = 1024 + (int)sizeof(WeightsSmem);
  const int rows = a.cols * D * 2, stages = (most - fixed - rows) / WT_PIECE;
  a.stages = stages < WT_STAGES ? stages : WT_STAGES;
  const int smem = fixed + rows + a.stages * WT_PIECE;
  static_assert(most - fixed - WT_ROWS * 512 >= 4 * WT_PIECE, "a ring beside the most queries");
  auto *kernel = &k_weights<D, F8>;
  static bool set[64];
  if (int rc = op_shared_memory(reinterpret_cast<const void *>(kernel), most, device, set)) return rc;
  const int64_t tiles = (int64_t)a.batch * a.heads * ((a.t + WT_KEYS - 1) / WT_KEYS);
  const unsigned grid = (unsigned)(tiles < sms ? tiles : sms);
  return op_cuda(op_launch(kernel, dim3(grid), dim3(WT_THREADS), smem, st, 1, map, a),
                 "k_weights launch");
}

template <bool F8>
int launch_weights_d(int d, const CUtensorMap &map, WeightsArgs &a, int sms, int device, cudaStream_t st) {
  if (d == 64) return launch_weights<64, F8>(map, a, sms, device, st);
  if (d == 128) return launch_weights<128, F8>(map, a, sms, device, st);
  return launch_weights<256, F8>(map, a, sms, device, st);
}

}  // namespace
}  // namespace skv

extern "C" int skv_accumulate_weights(const SkvWeights *d, void *stream) {
  using namespace skv;
  if (!d) return op_fail(SKV_E_INVALID, "null descriptor");
  if (d->dim != 64 && d->dim != 128 && d->dim != 256) return op_fail(SKV_E_INVALID, "head size must be 64, 128 or 256");
  if (d->kv_heads < 1 || d->heads < 1 || d->heads % d->kv_heads || d->heads > 4096)
    return op_fail(SKV_E_INVALID, "query heads must be a multiple of the KV heads, and at most 4096");
  if (d->batch < 0 || d->batch > (1 << 20) || d->n < 1 || d->n > INT32_MAX)
    return op_fail(SKV_E_INVALID, "batch must be in [0, 2^20], n in [1, 2^31)");
  if (d->tokens < 1 || d->tokens > (1 << 26)) return op_fail(SKV_E_INVALID, "tokens must be in [1, 2^26]");
  if (!(d->scale > 0.0) || !(d->scale < 1e30)) return op_fail(SKV_E_INVALID, "scale must be positive and finite");
  if (d->cache_dtype != SKV_DTYPE_BF16 && d->cache_dtype != SKV_DTYPE_E4M3)
    return op_fail(SKV_E_INVALID, "the cache is BF16 or FP8 e4m3");
  if (d->batch == 0) return SKV_OK;
  if (!d->q || !d->k_cache || !d->lengths || !d->lse || !d->weights || !d->weights_out)
    return op_fail(SKV_E_INVALID, "null input or output pointer");
  const bool f8 = d->cache_dtype == SKV_DTYPE_E4M3;
  const int64_t of_q[3] = {d->batch, d->n, d->heads}, of_cache[3] = {d->batch, d->kv_heads, d->tokens};
  int64_t qs[3], kcs[3], ws[3], os[3], ls[3];
  op_strides(qs, d->q_stride, of_q, 3);
  op_strides(kcs, d->k_cache_stride, of_cache, 3);
  op_strides(ws, d->weights_stride, of_cache, 3);
  op_strides(os, d->weights_out_stride, of_cache, 3);
  op_strides(ls, d->lse_stride, of_q, 3);
  if (d->q_stride[3] != 1 || d->k_cache_stride[3] != 1)
    return op_fail(SKV_E_INVALID, "the innermost dimension must be contiguous");
  bool ok = (uintptr_t)d->q % 16 == 0 && (uintptr_t)d->k_cache % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && qs[i] >= 0 && qs[i] % 8 == 0 && kcs[i] >= 0 && kcs[i] % (f8 ? 16 : 8) == 0;
  if (!ok) return op_fail(SKV_E_INVALID, "rows must start on 16-byte boundaries");
  if (d->tokens > 1 && !kcs[2]) return op_fail(SKV_E_INVALID, "tokens must not share one row");
  int sms = 0;
  if (int rc = sm_count(d->device, &sms)) return rc;
  DeviceScope scope((int)d->device);
  if (int rc = op_cuda(scope.error(), "selecting the device")) return rc;
  WeightsArgs a{};
  if (int rc = status_word((int)d->device, &a.status)) return rc;
  const int group = (int)(d->heads / d->kv_heads);
  a.heads = (int)d->kv_heads, a.group = group, a.t = (int)d->tokens;
  a.by_group = ((1ull << 32) + group - 1) / group;
  a.scale = (float)d->scale;
  a.len_stride = d->batch == 1 ? 0 : d->lengths_stride;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = qs[i], a.ls[i] = ls[i];
    a.os[i] = os[i];
  }
  op_strides(a.ts, d->rows_stride, of_q, 2);
  const int64_t rows = d->n * group;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t b0 = 0; b0 < d->batch; b0 += PLAN_BATCH) {
    const int64_t nb = d->batch - b0 < PLAN_BATCH ? d->batch - b0 : PLAN_BATCH;
    a.batch = (int)nb;
    a.lengths = static_cast<const int32_t *>(d->lengths) + b0 * a.len_stride;
    a.out = static_cast<float *>(d->weights_out) + b0 * a.os[0];
    CUtensorMap map{};
    const int64_t step[3] = {kcs[2], kcs[1], kcs[0]};
    const uint8_t *base = static_cast<const uint8_t *>(d->k_cache) + b0 * kcs[0] * (f8 ? 1 : 2);
    if (int rc = f8 ? make_byte_map(&map, base, d->dim, d->tokens, d->kv_heads, nb, step, WT_KEYS, d->dim == 64 ? 64 : 128, true)
                    : make_map(&map, base, d->dim, d->tokens, d->kv_heads, nb, step, WT_KEYS, 1))
      return rc;
    a.along[0] = kcs[1] ? 1 : 0;
    a.along[1] = nb > 1 && kcs[0] ? 1 : 0;
    // more rows than the MMA's N: further launches add to what the first wrote
    for (int64_t r0 = 0; r0 < rows; r0 += WT_ROWS) {
      // (from the node that holds row r0 on, so that the kernel's row numbers stay small)
      const int64_t node0 = r0 / group;
      a.q = static_cast<const uint16_t *>(d->q) + b0 * a.qs[0] + node0 * a.qs[1];
      a.lse = static_cast<const float *>(d->lse) + b0 * a.ls[0] + node0 * a.ls[1];
      a.take = d->rows ? static_cast<const uint8_t *>(d->rows) + b0 * a.ts[0] + node0 * a.ts[1] : nullptr;
      a.row0 = (int)(r0 - node0 * group);
      a.rows = (int)(rows - r0 < WT_ROWS ? rows - r0 : WT_ROWS);
      a.cols = (a.rows + 15) & ~15;
      if (r0 == 0) {
        a.w = static_cast<const float *>(d->weights) + b0 * ws[0];
        for (int i = 0; i < 3; ++i) a.ws[i] = ws[i];
      } else {
        a.w = a.out;
        for (int i = 0; i < 3; ++i) a.ws[i] = a.os[i];
      }
      const int rc = f8 ? launch_weights_d<true>((int)d->dim, map, a, sms, (int)d->device, st) : launch_weights_d<false>((int)d->dim, map, a, sms, (int)d->device, st);
      if (rc) return rc;
    }
  }
  return SKV_OK;
}
