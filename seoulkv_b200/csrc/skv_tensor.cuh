// skv_tensor.cuh -- the Blackwell tensor core, tensor memory, TMA and mbarrier
// instructions that the attention operators use, and waits that end.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/seoulkv_b200.h"

namespace skv {

__device__ __forceinline__ uint32_t s_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// The loading and the tensor-core warp run their loops as whole warps, and
// only their instructions are predicated on one elected lane: descriptors and
// addresses then stay in uniform registers.  In a branch that one lane takes,
// every instruction moves its operands there first, and the issue alone takes
// longer than the tensor core (2990 cycles against 2100 for a tile of 128 keys
// at D = 256, and 4200 beside busy warps).
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}

// ---- mbarriers -----------------------------------------------------------

// A wait that lasts WAIT_NS gives up: it raises `abort` for its CTA (every
// later wait then gives up at once, so that all roles run to their end
// without waiting) and a bit in the device's status word, which the host reads.
constexpr unsigned long long WAIT_NS = 2000000000ull;
constexpr int WAIT_FREE_POLLS = 256;

__device__ __forceinline__ unsigned long long timer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s_addr(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(s_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
static __device__ __noinline__ bool bar_wait_long(uint64_t *bar, uint32_t parity, volatile uint32_t *abort, uint32_t *status) {
  const unsigned long long t0 = timer_ns();
  do {
    for (int i = 0; i < WAIT_FREE_POLLS; ++i)
      if (bar_try(bar, parity)) return true;
    if (*abort) return false;
  } while (timer_ns() - t0 < WAIT_NS);
  *abort = 1;
  atomicOr(status, SKV_STATUS_TIMEOUT);
  return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort, uint32_t *status) {
  if (bar_try(bar, parity)) return true;
  return bar_wait_long(bar, parity, abort, status);
}

// Writes to shared memory by threads, before the tensor core or TMA reads them.
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- TMA (own memory, no multicast) ---------------------------------------

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// By the elected lane, before it loads with a map in global memory: what the
// host wrote there is what the load sees.  (A map that an earlier launch used
// at the same address may still be held by the SM.  Maps that are kernel
// parameters need none of this.)
__device__ __forceinline__ void tma_acquire_map(uint32_t one, const CUtensorMap *map) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q fence.proxy.tensormap::generic.acquire.sys [%0], 128;\n\t}" ::"l"(map),
      "r"(one)
      : "memory");
}
// The elected lane announces `bytes` on `bar` and loads the box at (row,
// piece, y, z) of a make_map() map.
__device__ __forceinline__ void tma_load(uint32_t one, void *dst, const CUtensorMap *map, int row, int piece, int y,
                                         int z, uint64_t *bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %8, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%7], %9;\n\t"
      "@q cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];\n\t}" ::"r"(s_addr(dst)),
      "l"(map), "r"(0), "r"(row), "r"(piece), "r"(y), "r"(z), "r"(s_addr(bar)), "r"(one), "r"(bytes)
      : "memory");
}

// The elected lane announces `bytes` on `bar` and loads the box at (byte, row,
// y, z) of a make_byte_map() map.
__device__ __forceinline__ void tma_load_bytes(uint32_t one, void *dst, const CUtensorMap *map, int byte, int row, int y,
                                               int z, uint64_t *bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %7, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%6], %8;\n\t"
      "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];\n\t}" ::"r"(s_addr(dst)),
      "l"(map), "r"(byte), "r"(row), "r"(y), "r"(z), "r"(s_addr(bar)), "r"(one), "r"(bytes)
      : "memory");
}

// ---- tensor memory and tcgen05.mma ----------------------------------------

__device__ __forceinline__ void tmem_alloc(uint32_t *where, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(where)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Arrives on `bar` when every MMA issued so far by the elected lane has ended.
__device__ __forceinline__ void mma_commit(uint32_t one, uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(s_addr(bar)),
      "r"(one)
      : "memory");
}

// Instruction descriptor: FP32 accumulator, BF16 operands, A K-major, B
// K-major or (b_rows) stored with its N index contiguous.
__host__ __device__ constexpr uint32_t mma_desc(int m, int n, bool b_rows) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
// Shared-memory operand in 128-byte-swizzled rows (8-row groups of 1024
// bytes); `lead` is the stride between 64-element pieces of an operand whose
// M or N index is contiguous (unused otherwise).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// FP32 accumulator, FP8 e4m3 operands, both K-major (a step is 32 codes).
__host__ __device__ constexpr uint32_t mma_desc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// K-major operand in rows of 128 or 64 bytes, swizzled over as many.
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t addr, int row_bytes) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | (1ull << 16) | ((uint64_t)(row_bytes * 8 >> 4) << 32) | (1ull << 46) |
         ((row_bytes == 128 ? 2ull : 4ull) << 61);
}
// The 16-byte unit of a swizzled row that holds its unit c.
__device__ __forceinline__ int swizzled(int c, int row, int row_bytes) {
  return row_bytes == 128 ? c ^ (row & 7) : c ^ (row >> 1 & 3);
}
// By the elected lane: D (tensor memory) = A B (shared memory, FP8) [+ D], K = 32.
__device__ __forceinline__ void mma_f8(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add), "r"(one)
      : "memory");
}
// By the elected lane: D (tensor memory) = A (tensor memory) B (shared memory) [+ D], K = 16.
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add), "r"(one)
      : "memory");
}
// By the elected lane: D (tensor memory) = A (shared memory) B (shared memory) [+ D], K = 16.
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add), "r"(one)
      : "memory");
}

#define SKV_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), \
                     "=r"(v[i + 6]), "=r"(v[i + 7])
#define SKV_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), \
                     "r"(v[i + 6]), "r"(v[i + 7])
// 32 / 16 consecutive columns of this thread's lane (warp w of four: lanes 32w..32w+31).
__device__ __forceinline__ void tmem_ld32(uint32_t (&v)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : SKV_R8(v, 0), SKV_R8(v, 8), SKV_R8(v, 16), SKV_R8(v, 24)
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&v)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : SKV_R8(v, 0), SKV_R8(v, 8)
      : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::SKV_W8(
          v, 0),
      SKV_W8(v, 8), "r"(at)
      : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
// 16 FP8 e4m3 codes to BF16, exactly.  The conversion instructions run at 16
// lanes a cycle and would take longer than the product that follows (8192
// codes: 1024 cycles of an SM), so the bits are moved instead: sign, exponent
// and mantissa of a code, put at a BF16's places, are its value times 2^-120
// (subnormal codes are subnormal there too), and the product with 2^120 is
// exact.  The one code that is not a number comes out as 480 and is put right
// where a piece has one.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t x, uint32_t pick) {
  // (pick: two bytes, each with its sign spread over the byte above)
  uint32_t bits, y;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(bits) : "r"(x), "r"(pick));
  bits = (bits << 4) & 0x87f087f0u;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(bits), "r"(0x7b807b80u));
  return y;
}
// (nan: one of bits 7, 15, 23, 31 is raised where a code is not a number: one
// more turns its sign bit, as the carry out of such a code may turn the next)
__device__ __forceinline__ void e4m3_to_bf16(const uint4 &x, uint4 &lo, uint4 &hi, uint32_t &nan) {
  lo = make_uint4(e4m3_pair(x.x, 0x9180), e4m3_pair(x.x, 0xb3a2), e4m3_pair(x.y, 0x9180), e4m3_pair(x.y, 0xb3a2));
  hi = make_uint4(e4m3_pair(x.z, 0x9180), e4m3_pair(x.z, 0xb3a2), e4m3_pair(x.w, 0x9180), e4m3_pair(x.w, 0xb3a2));
  nan |= x.x ^ (x.x + 0x01010101u);
  nan |= x.y ^ (x.y + 0x01010101u);
  nan |= x.z ^ (x.z + 0x01010101u);
  nan |= x.w ^ (x.w + 0x01010101u);
}
constexpr uint32_t E4M3_NAN = 0x80808080u;
// 480 to NaN, in 16 bytes that e4m3_to_bf16 wrote.
static __device__ __noinline__ void e4m3_put_nan(uint4 *at) {
  uint32_t *y = reinterpret_cast<uint32_t *>(at);
  for (int i = 0; i < 4; ++i) {
    if ((y[i] & 0x7fffu) == 0x43f0u) y[i] |= 0x7fffu;
    if ((y[i] & 0x7fff0000u) == 0x43f00000u) y[i] |= 0x7fff0000u;
  }
}
// ---- a BF16 row as the sum of two FP8 e4m3 rows
//
// A query q (8 significant bits) times 2^e, with e so that the row's largest
// element lies in [128, 256), is hi + lo: hi the nearest e4m3 (4 bits), lo what
// is left (a multiple of 2^-7 of hi's power of two, at most 2^-4 of it: 4 bits
// again).  The sum is exact wherever lo is no smaller than e4m3's last place,
// 2^-9: for elements above 2^-9 of the largest.  Below, it is off by half a
// last place, at most 2^-17 of the largest.  K in FP8 then goes to the tensor
// core as it is stored, twice (at twice the BF16 rate), instead of through
// registers into BF16.
//
// 2^e of a row that `lanes` neighbouring threads hold in 16-byte pieces, as
// the exponent field of a float (127: a row of zeros or not finite).
__device__ __forceinline__ uint32_t split_exponent(const uint4 &v, int lanes) {
  uint32_t top = 0;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, w[i] >> 16 & 0x7fffu));
  for (int o = lanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = (int)(top >> 7);  // the exponent field of BF16 and of FP32
  return top == 0 || e == 255 ? 127u : (uint32_t)min(261 - e, 253);
}
// Two elements (BF16 pair) times f: hi and lo codes, two bytes each.
__device__ __forceinline__ void split_pair(uint32_t pair, float f, uint32_t &hi, uint32_t &lo) {
  float x = __uint_as_float(pair << 16) * f, y = __uint_as_float(pair & 0xffff0000u) * f;
  x = isinf(x) ? __uint_as_float(0x7fffffffu) : x;  // (e4m3 has no infinity: a row with one is not a number)
  y = isinf(y) ? __uint_as_float(0x7fffffffu) : y;
  uint16_t h, l;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(y), "f"(x));
  uint32_t back;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h));
  float hx, hy;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(hx), "=f"(hy)
      : "r"(back));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(l) : "f"(y - hy), "f"(x - hx));
  hi = h;
  lo = l;
}
// Eight elements: eight bytes of hi, eight of lo.
__device__ __forceinline__ void split_eight(const uint4 &v, float f, uint2 &hi, uint2 &lo) {
  uint32_t h[4], l[4];
  split_pair(v.x, f, h[0], l[0]);
  split_pair(v.y, f, h[1], l[1]);
  split_pair(v.z, f, h[2], l[2]);
  split_pair(v.w, f, h[3], l[3]);
  hi = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  lo = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(lo), "f"(hi));
  return y;
}
__device__ __forceinline__ void unpack2(uint64_t x, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
// Two FP32 operations in one instruction.
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}

// ---- cp.async --------------------------------------------------------------

// 16 bytes to shared memory, zeros where !valid (nothing is read then).
__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s_addr(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---- host: tensor maps and the status word (skv_tree.cu) -------------------

// Map of [z][y][rows][dim] 16-bit elements with element strides {row, y, z},
// taken as pieces of 64 elements: a box is `box_rows` rows of `pieces` pieces,
// in shared memory piece after piece, each a stack of 128-byte rows with the
// 128-byte swizzle.  A dimension of one element, or of stride 0, is mapped
// with one element.
int make_map(CUtensorMap *map, const void *base, int64_t dim, int64_t rows, int64_t ny, int64_t nz,
             const int64_t *stride, int box_rows, int pieces);
// Map of [z][y][rows][bytes] with byte strides {row, y, z}, boxes of box_rows
// rows of box_bytes bytes one after the other (`swizzle`: swizzled over a
// row's 128 or 64 bytes).
int make_byte_map(CUtensorMap *map, const void *base, int64_t bytes, int64_t rows, int64_t ny, int64_t nz,
                  const int64_t *stride, int box_rows, int box_bytes, bool swizzle);
// The device's status word (set by waits that gave up).
int status_word(int device, uint32_t **word);

}  // namespace skv
