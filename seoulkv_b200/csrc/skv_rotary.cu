// skv_rotary.cu -- rotary positions on queries and keys.
//
// Pair i of a head's first R dimensions is turned by the angle p * f_i, with p
// the token's position and f_i the pair's frequency (radians per position):
//   half:        pair i = (x[i], x[i + R/2])
//   interleaved: pair i = (x[2i], x[2i + 1])
//   y_a = m (x_a cos - x_b sin),  y_b = m (x_a sin + x_b cos),
// and dimensions R.. are copied.  One read and one write of q and k.
//
// The angle.  p * f_i in FP32 is useless far out (at p = 2^20 it is off by
// 2^-4 rad).  f_i / 2 pi arrives as a 64-bit fraction of a turn, rounded once
// from more digits; the 64-bit product with the integer position keeps the
// fraction of a turn modulo one exactly, so there is no range reduction and the
// error is p * 2^-65 turns, negative positions included: below the rounding to
// FP32 that follows (2^-26 turns) up to p = 2^39.  The top 32 bits go to
// sincospif.
//
// Measured (a copy moves 6437 GB/s): 65536 tokens, 16 + 4 heads of 256 in FP32,
// 410 us for 2.68 GB, the copy rate: a token's sines are computed once for all
// of its heads.  One token, or 64 x 13 drafted ones in BF16 (17 MB, 2.6 us of
// traffic), 11.6 us a call: the host's time (2.6 and 7.4 us on the device).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <utility>

#include "skv_ops.cuh"

namespace skv {
namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_PAIRS = SKV_ROTARY_MAX_PAIRS;
constexpr int RT_UNROLL = 4;  // heads whose loads are in flight together

struct RotaryArgs {
  const void *x[2];     // q, k
  void *y[2];
  int64_t xs[2][3], ys[2][3];  // element strides (batch, token, head)
  const void *positions;
  int64_t pos_stride[2];  // (batch, token)
  int64_t tokens;       // batch * n
  int n, heads[2], dim, pairs, pos64;
  int chunks, rot_chunks;  // per head: all work items, and those that rotate
  int split;            // threads that share a token's heads
  float m;
  uint64_t phase[RT_PAIRS];  // turns per position * 2^64
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// One thread: V elements of each of a pair's two places (half), or V
// consecutive elements (interleaved, and the dimensions that are copied), of
// heads s, s + split, ... of one token.  Its sines serve all of its heads.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(RT_THREADS) k_rotary(const __grid_constant__ RotaryArgs a) {
  // lanes need different pairs: from shared memory (the parameter bank would
  // serve a warp's 32 addresses one by one, at every use)
  __shared__ uint64_t s_phase[RT_PAIRS];
  for (int i = threadIdx.x; i < a.pairs; i += RT_THREADS) s_phase[i] = a.phase[i];
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_release();
  constexpr int NP = HALF ? V : (V + 1) / 2;  // pairs of one thread
  using W = Vec<T, V>;
  const int64_t items = a.tokens * a.split * a.chunks;
  const int total = a.heads[0] + a.heads[1];
  const int half = a.pairs;
  for (int64_t it = (int64_t)blockIdx.x * RT_THREADS + threadIdx.x; it < items;
       it += (int64_t)gridDim.x * RT_THREADS) {
    const int c = (int)(it % a.chunks);
    const int64_t r = it / a.chunks;
    const int s = (int)(r % a.split);
    const int64_t tok = r / a.split;
    const int64_t b = tok / a.n, t = tok - b * a.n;
    const bool rot = c < a.rot_chunks;
    const int d0 = rot || !HALF ? c * V : 2 * half + (c - a.rot_chunks) * V;
    float cs[NP], sn[NP];
    if (rot) {
      const int64_t po = b * a.pos_stride[0] + t * a.pos_stride[1];
      const int64_t p = a.pos64 ? static_cast<const int64_t *>(a.positions)[po]
                                : static_cast<const int32_t *>(a.positions)[po];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int pair = HALF ? d0 + j : d0 / 2 + j;
        const uint64_t turn = (uint64_t)p * s_phase[pair];
        // the top 32 bits as a signed fraction of a turn: 2^-31 half turns
        sincospif((float)(int32_t)(uint32_t)(turn >> 32) * 4.656612873077393e-10f, &sn[j], &cs[j]);
        sn[j] *= a.m;
        cs[j] *= a.m;
      }
    }
    for (int h0 = s; h0 < total; h0 += a.split * RT_UNROLL) {
      W lo[RT_UNROLL], hi[RT_UNROLL];
#pragma unroll
      for (int u = 0; u < RT_UNROLL; ++u) {
        const int h = h0 + u * a.split;
        if (h >= total) break;
        const int w = h >= a.heads[0];
        const T *x = static_cast<const T *>(a.x[w]) + b * a.xs[w][0] + t * a.xs[w][1] +
                     (h - (w ? a.heads[0] : 0)) * a.xs[w][2] + d0;
        lo[u] = *reinterpret_cast<const W *>(x);
        if (HALF && rot) hi[u] = *reinterpret_cast<const W *>(x + half);
      }
#pragma unroll
      for (int u = 0; u < RT_UNROLL; ++u) {
        const int h = h0 + u * a.split;
        if (h >= total) break;
        const int w = h >= a.heads[0];
        T *y = static_cast<T *>(a.y[w]) + b * a.ys[w][0] + t * a.ys[w][1] + (h - (w ? a.heads[0] : 0)) * a.ys[w][2] +
               d0;
        if (rot) {
          if (HALF) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float p = to_f(lo[u].v[j]), q = to_f(hi[u].v[j]);
              lo[u].v[j] = from_f<T>(p * cs[j] - q * sn[j]);
              hi[u].v[j] = from_f<T>(p * sn[j] + q * cs[j]);
            }
            *reinterpret_cast<W *>(y + half) = hi[u];
          } else {
#pragma unroll
            for (int j = 0; j + 1 < V; j += 2) {
              const float p = to_f(lo[u].v[j]), q = to_f(lo[u].v[j + 1]);
              lo[u].v[j] = from_f<T>(p * cs[j / 2] - q * sn[j / 2]);
              lo[u].v[j + 1] = from_f<T>(p * sn[j / 2] + q * cs[j / 2]);
            }
          }
        }
        *reinterpret_cast<W *>(y) = lo[u];
      }
    }
  }
}

template <typename T, int V>
cudaError_t launch_rotary(const RotaryArgs &a, bool half, int sms, cudaStream_t st) {
  const int64_t items = a.tokens * a.split * a.chunks;
  const int64_t want = (items + RT_THREADS - 1) / RT_THREADS;
  const unsigned grid = (unsigned)(want < 16LL * sms ? want : 16LL * sms);
  if (half) return op_launch(k_rotary<T, V, true>, dim3(grid), dim3(RT_THREADS), 0, st, 1, a);
  return op_launch(k_rotary<T, V < 2 ? 2 : V, false>, dim3(grid), dim3(RT_THREADS), 0, st, 1, a);
}

template <typename T>
cudaError_t launch_rotary_v(const RotaryArgs &a, bool half, int v, int sms, cudaStream_t st) {
  if (v * sizeof(T) >= 16) return launch_rotary<T, 16 / sizeof(T)>(a, half, sms, st);
  if (v >= 4) return launch_rotary<T, 4>(a, half, sms, st);
  if (v == 2) return launch_rotary<T, 2>(a, half, sms, st);
  return launch_rotary<T, 1>(a, half, sms, st);
}

}  // namespace
}  // namespace skv

extern "C" int skv_rotary(const SkvRotary *d, void *stream) {
  using namespace skv;
  if (!d) return op_fail(SKV_E_INVALID, "null descriptor");
  const bool has_k = d->kv_heads > 0;
  if (d->batch < 0 || d->n < 0 || d->heads < 1 || d->kv_heads < 0 || d->batch > INT32_MAX || d->n > INT32_MAX ||
      d->heads > 65535 || d->kv_heads > 65535)
    return op_fail(SKV_E_INVALID, "batch, n or head counts out of range");
  if (d->dim < 2 || d->dim > 65536 || d->rotary_dim < 2 || d->rotary_dim % 2 || d->rotary_dim > d->dim ||
      d->rotary_dim / 2 > RT_PAIRS)
    return op_fail(SKV_E_INVALID, "rotary_dim must be even, in [2, min(dim, %d)]", 2 * RT_PAIRS);
  if (d->dtype < SKV_DTYPE_BF16 || d->dtype > SKV_DTYPE_FP32) return op_fail(SKV_E_INVALID, "q and k are BF16, FP16 or FP32");
  if (d->layout != SKV_ROTARY_HALF && d->layout != SKV_ROTARY_INTERLEAVED)
    return op_fail(SKV_E_INVALID, "unknown rotary layout");
  if (d->batch == 0 || d->n == 0) return SKV_OK;
  if (d->q_stride[3] != 1 || d->q_out_stride[3] != 1 || (has_k && (d->k_stride[3] != 1 || d->k_out_stride[3] != 1)))
    return op_fail(SKV_E_INVALID, "the innermost dimension must be contiguous");
  if (!d->q || !d->q_out || (has_k && (!d->k || !d->k_out)) || !d->positions || !d->phase)
    return op_fail(SKV_E_INVALID, "null input or output pointer");
  int sms = 0;
  if (int rc = sm_count(d->device, &sms)) return rc;
  DeviceScope scope((int)d->device);
  if (int rc = op_cuda(scope.error(), "selecting the device")) return rc;
  const bool half = d->layout == SKV_ROTARY_HALF;
  const int size = d->dtype == SKV_DTYPE_FP32 ? 4 : 2;
  RotaryArgs a;
  a.x[0] = d->q, a.x[1] = d->k, a.y[0] = d->q_out, a.y[1] = d->k_out;
  const int64_t nq[3] = {d->batch, d->n, d->heads}, nk[3] = {d->batch, d->kv_heads, d->n};
  op_strides(a.xs[0], d->q_stride, nq, 3);
  op_strides(a.ys[0], d->q_out_stride, nq, 3);
  op_strides(a.xs[1], d->k_stride, nk, 3);
  op_strides(a.ys[1], d->k_out_stride, nk, 3);
  std::swap(a.xs[1][1], a.xs[1][2]);  // (batch, token, head) as q's
  std::swap(a.ys[1][1], a.ys[1][2]);
  a.positions = d->positions;
  a.pos64 = d->pos64 != 0;
  op_strides(a.pos_stride, d->pos_stride, nq, 2);
  a.tokens = d->batch * d->n;
  a.n = (int)d->n;
  a.heads[0] = (int)d->heads, a.heads[1] = (int)d->kv_heads;
  a.dim = (int)d->dim;
  a.pairs = (int)d->rotary_dim / 2;
  a.m = (float)d->factor;
  memcpy(a.phase, d->phase, sizeof(uint64_t) * a.pairs);
  // the widest access (16 bytes down to one element) that every row start,
  // the rotated part's halves and the copied rest allow
  int v = 16 / size;
  auto fits = [&](int w) {
    if (half ? a.pairs % w : (2 * a.pairs) % w) return false;
    if (a.dim % w) return false;
    for (int i = 0; i < (has_k ? 2 : 1); ++i) {
      if ((uintptr_t)a.x[i] % (w * size) || (uintptr_t)a.y[i] % (w * size)) return false;
      for (int j = 0; j < 3; ++j)
        if (a.xs[i][j] % w || a.ys[i][j] % w) return false;
    }
    return true;
  };
  while (v > 1 && !fits(v)) v /= 2;
  if (!half && v < 2) v = 2;  // an interleaved pair is one access of two elements ...
  if (!half && !fits(v))      // ... so its pairs have to be aligned to themselves
    return op_fail(SKV_E_INVALID, "interleaved pairs must be aligned to two elements (head_dim and strides even)");
  if (half) {
    a.rot_chunks = a.pairs / v;
    a.chunks = a.rot_chunks + (a.dim - 2 * a.pairs) / v;
  } else {
    a.rot_chunks = 2 * a.pairs / v;
    a.chunks = a.dim / v;
  }
  // few tokens: more threads share a token's heads (each computes its own
  // sines); many tokens: one thread per token and chunk, sines computed once
  const int total = a.heads[0] + a.heads[1];
  const int64_t per = a.tokens * a.chunks;
  int64_t split = (1024LL * sms + per - 1) / per;
  a.split = (int)(split < 1 ? 1 : split > total ? total : split);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = d->dtype == SKV_DTYPE_FP32   ? launch_rotary_v<float>(a, half, v, sms, st)
                  : d->dtype == SKV_DTYPE_BF16 ? launch_rotary_v<__nv_bfloat16>(a, half, v, sms, st)
                                               : launch_rotary_v<__half>(a, half, v, sms, st);
  return op_cuda(e, "k_rotary launch");
}
