// Blackwell building blocks of the attention kernels: bounded mbarrier waits, TMA tile loads,
// tcgen05 matrix products with accumulators (and left operands) in tensor memory.
//
// Tiles in shared memory are rows of 64 16-bit elements (128 bytes) in the 128-byte swizzle that
// TMA writes: the 16-byte chunk c of row r lies at chunk c ^ (r & 7).  A tile of 128 rows
// and a head size above 64 is two such blocks, one after the other; so are tiles of 64 rows.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace b3r {

constexpr int kTileRows = 128;
constexpr int kBlockBytes = kTileRows * 128;   // 128 rows of 64 elements

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarriers.  No wait is endless: after its limit it raises `dead`, which ends the later
// waits of every role soon; the loops all have fixed counts, so the kernel then runs to its
// end, frees its tensor memory and reports the failure.  What a failed wait was for is not done: no copy to a
// barrier whose last one is still out, no job over one in use.  Lanes see `dead` at different times, so a warp
// votes on it, and groups of warps meet on mbarriers alone, never on counted barriers after a choice.
__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.shared::cta.b64 t, [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
constexpr int kWaitLimit = 1 << 18;   // polls of 4 us: measured, 1.04 s until a wait runs out, where one takes microseconds
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* dead, int limit = kWaitLimit) {
  if (mbar_try(bar, parity)) return true;
  for (int n = 0; n < limit; ++n) {
    if (mbar_try(bar, parity)) return true;
    if ((n & 63) == 63 && *dead) return false;   // (every poll: 4 % of the attention kernels)
  }
  *dead = 1;
  return false;
}

// ---- TMA: one box of 64 elements x some rows of a (D, rows, heads, batch) tensor
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int d0, int row, int head, int batch, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(d0), "r"(row), "r"(head), "r"(batch), "r"(bar)
      : "memory");
}
// An untiled copy of `bytes` (a multiple of 16, both addresses 16-byte aligned).
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tcgen05
__device__ __forceinline__ void tc_alloc(uint32_t where, int cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tc_free(uint32_t tmem, int cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// One lane of a converged warp.  The issuing warp stays converged, with uniform operands, and
// this lane's predicate on the instructions themselves: issued from within a branch of one lane each
// product took 75 to 140 cycles to issue, more than the tensor cores need for it.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on;
}
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(on)
      : "memory");
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((int)acc), "r"(on)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]: row i of A in lane i, two elements to a column
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((int)acc), "r"(on)
      : "memory");
}

// Shared-memory operand descriptors (128-byte swizzle).
// k-major: the product runs along the 64 elements of a row; 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// mn-major: the product runs along the rows (8-row groups 1024 bytes apart); blocks of 64
// elements of the other dimension lie `block` bytes apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, int block) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t(block >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// One step of 16, k-major without swizzle: bricks of 8 rows x 16 bytes, the step's two side by side, 8-row
// groups 256 bytes apart.
__device__ __forceinline__ uint64_t desc_step(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t(128 >> 4) << 16) | (uint64_t(256 >> 4) << 32) | (uint64_t(1) << 46);
}
// Instruction descriptor: float32 accumulator, both operands bf16 or both f16.
__host__ __device__ constexpr uint32_t mma_idesc(bool bf16, int M, int N, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// tile_product: acc = A B^T over the head size in `steps` steps of 16; A has 128 rows, B has ROWS, both k-major.
// tile_gather: acc (+)= A B over the ROWS rows of tile b; A in tensor memory, its first 64 rows' steps
// from `a`, the others' from `a + half`.  Offsets within a tile only change the descriptors' address field
// (units of 16 bytes).
template <int BLOCKS, int ROWS>
__device__ __forceinline__ void tile_product(uint32_t acc, uint32_t a, uint32_t b, uint32_t idesc, int steps, uint32_t on) {
  const uint64_t da = desc_k(a), db = desc_k(b);
#pragma unroll
  for (int t = 0; t < BLOCKS * 4; ++t)
    if (t < steps)
      tc_mma(acc, da + (((t >> 2) * kBlockBytes + (t & 3) * 32) >> 4), db + (((t >> 2) * ROWS * 128 + (t & 3) * 32) >> 4), idesc, t > 0,
             on);
}
// The same with A in tensor memory (two elements to a column): a left operand in shared memory costs about 100
// cycles for 16 of the head size, one in tensor memory the 64 that the product takes.
template <int BLOCKS, int ROWS>
__device__ __forceinline__ void tile_product_ts(uint32_t acc, uint32_t a, uint32_t b, uint32_t idesc, int steps, uint32_t on) {
  const uint64_t db = desc_k(b);
#pragma unroll
  for (int t = 0; t < BLOCKS * 4; ++t)
    if (t < steps) tc_mma_ts(acc, a + t * 8, db + (((t >> 2) * ROWS * 128 + (t & 3) * 32) >> 4), idesc, t > 0, on);
}
template <int ROWS>
__device__ __forceinline__ void tile_gather(uint32_t acc, uint32_t a, int half, uint32_t b, uint32_t idesc, bool add, uint32_t on) {
  const uint64_t db = desc_mn(b, ROWS * 128);
#pragma unroll
  for (int t = 0; t < ROWS / 16; ++t) tc_mma_ts(acc, a + (t >> 2) * half + (t & 3) * 8, db + (t * 2048 >> 4), idesc, add || t > 0, on);
}

#define B3R_R4(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3])
#define B3R_R16(a, i) B3R_R4(a, i), B3R_R4(a, i + 4), B3R_R4(a, i + 8), B3R_R4(a, i + 12)
#define B3R_W4(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3])
#define B3R_W16(a, i) B3R_W4(a, i), B3R_W4(a, i + 4), B3R_W4(a, i + 8), B3R_W4(a, i + 12)

// 32 columns of this thread's lane (the warp's quarter of the 128 lanes).  The registers hold the
// values only after tc_wait_ld().
__device__ __forceinline__ void tc_ld32(uint32_t tmem, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : B3R_R16(r, 0), B3R_R16(r, 16)
      : "r"(tmem));
}
__device__ __forceinline__ void tc_st32(uint32_t tmem, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::B3R_W16(r, 0),
      B3R_W16(r, 16), "r"(tmem)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t tmem, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::B3R_W16(
          r, 0),
      "r"(tmem)
      : "memory");
}
// Waits for this thread's loads.  The empty statements tie the registers' uses to after the wait.
template <int N>
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t x, __nv_bfloat16) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t x, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// ---- a ring of shared-memory stages, each one tile of rows, filled by one warp
struct Ring {
  uint32_t data;              // shared address of stage 0
  uint8_t* data_ptr;          // the same, as a pointer
  const uint64_t *full, *empty;
  int stages;
  int stage = 0, round = 0;

  __device__ __forceinline__ void step() {
    if (++stage == stages) {
      stage = 0;
      ++round;
    }
  }
  // Consumer: the stage with the next tile, once it is there.
  __device__ __forceinline__ int next(volatile int* dead) {
    mbar_wait(smem_u32(full + stage), round & 1, dead);
    const int s = stage;
    step();
    return s;
  }
};

// Producer (a whole warp): the next stage gets rows [row, row + ROWS) of a head.  Only `valid` of
// them belong to the sequence; the others are the neighbours' or padding, and may hold NaN.  They
// are cleared where `clear`: where they meet zeros in a product along the rows.
template <int BLOCKS, int ROWS>
__device__ __forceinline__ void ring_load(Ring& g, const CUtensorMap* map, int row, int head, int batch, int valid, bool clear,
                                          uint64_t* fix, int& fixes, int lane, volatile int* dead) {
  const uint32_t full = smem_u32(g.full + g.stage), bar_fix = smem_u32(fix);
  constexpr int kBytes = ROWS * 128;
  const int at = g.stage * BLOCKS * kBytes;
  const bool cut = clear && valid < ROWS;
  bool go = true;
  if (g.round > 0) go = mbar_wait(smem_u32(g.empty + g.stage), (g.round - 1) & 1, dead);
  if (cut) go = __all_sync(0xffffffffu, go && !*dead);     // (bar_fix is met at once, unless a wait has failed)
  if (lane == 0 && go) {
    const uint32_t bar = cut ? bar_fix : full;
    mbar_expect(bar, BLOCKS * kBytes);
#pragma unroll
    for (int c = 0; c < BLOCKS; ++c) tma_box(g.data + at + c * kBytes, map, c * 64, row, head, batch, bar);
  }
  if (cut && go) {
    mbar_wait(bar_fix, fixes & 1, dead);
    ++fixes;
    for (int i = max(valid, 0) * 8 + lane; i < ROWS * 8; i += 32)
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) *reinterpret_cast<uint4*>(g.data_ptr + at + c * kBytes + i * 16) = make_uint4(0, 0, 0, 0);
    fence_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(full);
  }
  g.step();
}

}  // namespace b3r
