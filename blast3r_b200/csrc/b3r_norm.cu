// Part 5 of the C ABI: the norms before and after a block, with the block's gate and residual scale.
//
//   n = N(y; w_post, b_post)  (or y),   r = alpha x + g n,   h = N(r; w_pre, b_pre)  (optional)
//
// N subtracts the row's mean (layer norm only), divides by sqrt(mean square + eps), and applies
// weight and bias.  Backward, with dr the gradient that reaches r past h:
//   z = dh w_pre,  dr' = dr + rstd (z - [mean z] - rhat mean(z rhat)),  dx = alpha dr',
//   dg = dr' n,  dn = dr' g,  dy = the same map of dn w_post with yhat;  dw = sum dn xhat, db = sum dn
// (the bracketed term for layer norm).  The statistics are recomputed from y and r, which the
// pass reads anyway, so the forward pass saves nothing.
//
// Every row is read once and written once, so HBM bounds both passes.  A row belongs to one
// group of threads that keeps it in registers from the loads to the stores; its sums are float32,
// over the row twice (mean, then squares about it), joined by shuffles and, for more than one
// warp, through shared memory.  Backward, a block walks over a contiguous run of rows with the
// next row's loads in flight, and keeps the column sums (dw, db, dg) in registers; it writes them
// once as a partial, and a second kernel adds the partials in a fixed order: no atomics, so the
// results do not change from run to run.
//
// Measured on one B200, where a copy moves 6.5 TB/s: forward, 49216 layer-norm rows of 1024, float32 stream and
// bfloat16 branch, 93 us (6.5 TB/s); backward, 32768 RMS rows of 4096, bfloat16, two norms and a gate, 382 us
// (4.2 TB/s) and 7 us for the partials.  There one block of 512 threads fills an SM's registers, so the
// latency of a row's sum, barrier included, is hidden by nothing but the copies of the next rows.  Rows
// that no vector divides take two to three times as long (forward: 18600 rows of 2647, 268 us).
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "b3r_status.h"
#include "b3r_tc.cuh"

namespace b3r {
namespace {

constexpr int kE = 8;        // consecutive elements of one vector access
constexpr int kP = kE / 2;   // in packed pairs
constexpr int kMaxStages = 4;   // rows of the backward pass's ring

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ld1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void st1(float* p, float x) { *p = x; }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void st1(__half* p, float x) { *p = __float2half_rn(x); }

__device__ __forceinline__ float2 unpack(uint32_t x, __nv_bfloat16) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t x, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint32_t pack(float2 x, __nv_bfloat16) {
  const __nv_bfloat162 t = __float22bfloat162_rn(x);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t pack(float2 x, __half) {
  const __half2 t = __float22half2_rn(x);
  return *reinterpret_cast<const uint32_t*>(&t);
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Eight elements as they lie in memory: 16 bytes, or 32 of float32.
template <typename T>
struct Raw8 {
  uint32_t v[kE * sizeof(T) / 4];
};

// One access of 16 or 32 bytes, past L1: every row is used once.
__device__ __forceinline__ void fetch8(Raw8<float>& d, const float* p) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(d.v[0]), "=r"(d.v[1]), "=r"(d.v[2]), "=r"(d.v[3]), "=r"(d.v[4]), "=r"(d.v[5]), "=r"(d.v[6]), "=r"(d.v[7])
               : "l"(p));
}
template <typename T>
__device__ __forceinline__ void fetch8(Raw8<T>& d, const T* p) {
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(d.v[0]), "=r"(d.v[1]), "=r"(d.v[2]), "=r"(d.v[3])
               : "l"(p));
}
__device__ __forceinline__ void put8(float* p, const float2 (&x)[kP]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(__float_as_uint(x[0].x)),
               "r"(__float_as_uint(x[0].y)), "r"(__float_as_uint(x[1].x)), "r"(__float_as_uint(x[1].y)),
               "r"(__float_as_uint(x[2].x)), "r"(__float_as_uint(x[2].y)), "r"(__float_as_uint(x[3].x)),
               "r"(__float_as_uint(x[3].y))
               : "memory");
}
template <typename T>
__device__ __forceinline__ void put8(T* p, const float2 (&x)[kP]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack(x[0], T()), pack(x[1], T()), pack(x[2], T()), pack(x[3], T()));
}
__device__ __forceinline__ void widen(float2 (&o)[kP], const Raw8<float>& d) {
#pragma unroll
  for (int j = 0; j < kP; ++j) o[j] = make_float2(__uint_as_float(d.v[2 * j]), __uint_as_float(d.v[2 * j + 1]));
}
template <typename T>
__device__ __forceinline__ void widen(float2 (&o)[kP], const Raw8<T>& d) {
#pragma unroll
  for (int j = 0; j < kP; ++j) o[j] = unpack(d.v[j], T());
}

// The columns of a thread: vector v holds columns (v * threads + tid) * 8 + j, in one access, or,
// where the row's length or an address does not allow vectors, (v * 8 + j) * threads + tid.
template <bool VEC>
__device__ __forceinline__ int col_of(int v, int j, int tid, int threads) {
  return VEC ? (v * threads + tid) * kE + j : (v * kE + j) * threads + tid;
}

// A vector of a row of T in float32; zeros past the row.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(float2 (&o)[kP], const T* p, int v, int tid, int threads, int C) {
  if constexpr (VEC) {
    Raw8<T> d{};
    const int c = (v * threads + tid) * kE;
    if (c < C) fetch8(d, p + c);
    widen(o, d);
  } else {
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      const int c0 = col_of<false>(v, 2 * j, tid, threads), c1 = col_of<false>(v, 2 * j + 1, tid, threads);
      o[j] = make_float2(c0 < C ? ld1(p + c0) : 0.f, c1 < C ? ld1(p + c1) : 0.f);
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float2 (&x)[kP], int v, int tid, int threads, int C) {
  if constexpr (VEC) {
    const int c = (v * threads + tid) * kE;
    if (c < C) put8(p + c, x);
  } else {
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      const int c0 = col_of<false>(v, 2 * j, tid, threads), c1 = col_of<false>(v, 2 * j + 1, tid, threads);
      if (c0 < C) st1(p + c0, x[j].x);
      if (c1 < C) st1(p + c1, x[j].y);
    }
  }
}

// A vector of a weight, bias or gate row, which is float32 or the activations' type.
template <typename T, bool VEC>
__device__ __forceinline__ void load_w(float2 (&o)[kP], const void* p, bool f32, int v, int tid, int threads, int C) {
  if constexpr (VEC) {                             // cached: every row uses them
    const int c = (v * threads + tid) * kE;
#pragma unroll
    for (int j = 0; j < kP; ++j) o[j] = both(0.f);
    if (c >= C) return;
    if (f32) {
      const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + c);
      const float4 x = __ldg(q), y = __ldg(q + 1);
      o[0] = make_float2(x.x, x.y), o[1] = make_float2(x.z, x.w), o[2] = make_float2(y.x, y.y), o[3] = make_float2(y.z, y.w);
    } else if constexpr (sizeof(T) == 2) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p) + c));
      o[0] = unpack(x.x, T()), o[1] = unpack(x.y, T()), o[2] = unpack(x.z, T()), o[3] = unpack(x.w, T());
    }
  } else {
    if (f32) load8<float, false>(o, reinterpret_cast<const float*>(p), v, tid, threads, C);
    else load8<T, false>(o, reinterpret_cast<const T*>(p), v, tid, threads, C);
  }
}

// Whether the pair's columns lie in the row (1) or past it (0).
template <bool VEC>
__device__ __forceinline__ float2 inside(int v, int j, int tid, int threads, int C) {
  return make_float2(col_of<VEC>(v, 2 * j, tid, threads) < C ? 1.f : 0.f, col_of<VEC>(v, 2 * j + 1, tid, threads) < C ? 1.f : 0.f);
}

constexpr int kSums = 8;   // room for the values of one row_sum
template <int MAXW>
constexpr int kSumRow = MAXW == 32 ? 32 : 16;            // floats of a value's warps
template <int MAXW>
constexpr int kSumFloats = 2 * kSums * kSumRow<MAXW>;
// Sums of K values over the row's threads, by shuffles within a warp and through `buf` (two sets, used in
// turn, so one barrier per call is enough) over the warps, in a fixed order.  Two or
// more values share their shuffles: after a step that swaps them, half of the lanes go on with each.
template <int K, int MAXW>
__device__ __forceinline__ void row_sum(float (&s)[K], int warps, float* buf, int& turn) {
  static_assert(K == 1 || K == 2 || K == 3 || K == 6);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto swap = [&](float a, float b, int d) {           // lanes without bit d go on with a, the others with b
    const bool up = lane & d;
    return (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, d);
  };
  auto fold = [&](float a, int d) { return a + __shfl_xor_sync(0xffffffffu, a, d); };
  float v;
  constexpr int first = K == 1 ? 16 : K == 2 ? 8 : K == 3 ? 4 : 2;   // the distance at which one value a lane is left
  if constexpr (K == 1) {
    v = s[0];
  } else if constexpr (K == 2) {
    v = swap(s[0], s[1], 16);
  } else if constexpr (K == 3) {
    v = swap(swap(s[0], s[1], 16), fold(s[2], 16), 8);
  } else {
    v = swap(swap(swap(s[0], s[1], 16), swap(s[2], s[3], 16), 8), fold(swap(s[4], s[5], 16), 8), 4);
  }
#pragma unroll
  for (int d = first; d > 0; d >>= 1) v = fold(v, d);
  // value k ended up in the lanes whose bits 16, 8 and 4 are the bits 1, 2 and 4 of k
  if (warps == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = K == 1 ? v : __shfl_sync(0xffffffffu, v, (k & 1) * 16 + (k >> 1 & 1) * 8 + (k >> 2) * 4);
    return;
  }
  constexpr int kRow = kSumRow<MAXW>;                  // entries past the last warp stay zero
  float* b = buf + turn * kSums * kRow;
  turn ^= 1;
  const int mine = (lane >> 4) | (lane >> 2 & 2) | (lane & 4);
  if ((lane & (2 * first - 1)) == 0 && (K == 1 || mine < K)) b[(K == 1 ? 0 : mine) * kRow + w] = v;
  __syncthreads();
  if constexpr (MAXW == 32) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = b[k * kRow + lane];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) t = fold(t, d);
      s[k] = t;
    }
  } else {                                             // four lanes add up each value's row, four entries to a lane
    const float4 x = reinterpret_cast<const float4*>(b + (lane >> 2) * kRow)[lane & 3];
    const float t = fold(fold((x.x + x.y) + (x.z + x.w), 1), 2);
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = __shfl_sync(0xffffffffu, t, 4 * k);
  }
}
__device__ __forceinline__ void clear_sums(float* buf, int n) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) buf[i] = 0.f;
}

struct NormArgs {
  int64_t rows, rows_per_gate;
  int C, layer, wf32;            // wf32: weights, biases and gates are float32
  float eps, alpha;
  const void *y, *x, *dr, *dh;   // x: the stream forward, r backward
  int64_t y_row, x_row, dr_row, dh_row;
  const void *w_post, *b_post, *gate, *w_pre, *b_pre;
  void *r, *h, *dx, *dy;         // rows of C, contiguous
  float *part, *gpart;           // backward partials
  void* dgate;
  int post, pre, want_cols, gate_direct, stages, biases;
  int wait_limit, lose;         // backward: polls of a wait; for a test, copies of a block's last row are not asked for
  int32_t* status;
};

// Room for a row in shared memory.  Without VEC a row may begin anywhere: the whole 16-byte units that hold it
// are copied, and its place in the first one is kept.
template <typename T, bool VEC>
__host__ __device__ inline int slot_bytes(int C) {
  return VEC ? C * (int)sizeof(T) : (C * (int)sizeof(T) + 30) & ~15;
}

// ---------------------------------------------------------------- forward
// Rows that no vector divides pass through shared memory where they hold 16-bit elements, so that memory sees whole
// 16-byte units: 165230 rows of 701, float32 stream and bfloat16 branch, no norms, 248 us against 479 one element
// at a time; 18600 float16 rows of 2647 268 against 350.  Single float32 elements fill a warp's 128 bytes as
// they are (18600 rows of 7999: 641 us, through shared memory 755).
template <typename TY, bool VEC>
__host__ __device__ constexpr bool staged() {
  return !VEC && sizeof(TY) == 2;
}
// Where a row's first element lies in its slot.
template <typename T>
__device__ __forceinline__ T* in_slot(uint8_t* slot, const T* p) {
  return reinterpret_cast<T*>(slot + (reinterpret_cast<uintptr_t>(p) & 15));
}
template <typename T>
__device__ __forceinline__ void ask_row(uint8_t* slot, const T* p, int C, int tid, int threads) {
  const uint8_t* from = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
  const int end = (int)(reinterpret_cast<uintptr_t>(p) & 15) + C * (int)sizeof(T);
  for (int u = tid * 16; u < end; u += threads * 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slot + u)), "l"(from + u) : "memory");
}
template <typename T>
__device__ __forceinline__ void put_row(T* p, const uint8_t* slot, int C, int tid, int threads) {
  uint8_t* to = reinterpret_cast<uint8_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
  const int first = (int)(reinterpret_cast<uintptr_t>(p) & 15), end = first + C * (int)sizeof(T);
  for (int u = tid * 16; u < end; u += threads * 16) {
    if (u >= first && u + 16 <= end) {
      *reinterpret_cast<uint4*>(to + u) = *reinterpret_cast<const uint4*>(slot + u);
    } else {                                       // the unit's other bytes are another row's
      for (int e = max(u, first); e < min(u + 16, end); e += (int)sizeof(T))
        *reinterpret_cast<T*>(to + e) = *reinterpret_cast<const T*>(slot + e);
    }
  }
}

// POST: with a norm of y, y and x are both held until its statistics are known; without it, only r.
template <typename TX, typename TY, int VPT, bool VEC, bool POST>
__global__ void __launch_bounds__(256) k_norm_fwd(const __grid_constant__ NormArgs a) {
  constexpr bool kStage = staged<TY, VEC>();
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ alignas(16) float buf[kSumFloats<8>];
  // blockDim.x threads to a row; blocks of several rows have one warp to a row
  const int threads = blockDim.x, tid = threadIdx.x, warps = threads >> 5, C = a.C;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (warps > 1) {
    clear_sums(buf, kSumFloats<8>);
    __syncthreads();
  }
  if (row >= a.rows) return;                       // uniform over the row's threads
  int turn = 0;
  const TY* yp = reinterpret_cast<const TY*>(a.y) + row * a.y_row;
  const TX* xp = reinterpret_cast<const TX*>(a.x) + row * a.x_row;
  TX* rp = reinterpret_cast<TX*>(a.r) + row * C;
  TY* hp = reinterpret_cast<TY*>(a.h) + row * C;
  uint8_t *slot_x = nullptr, *slot_y = nullptr;
  auto meet = [&] {                                // the row's threads
    if (warps > 1) __syncthreads();
    else __syncwarp();
  };
  if constexpr (kStage) {
    slot_x = dyn + threadIdx.y * (slot_bytes<TX, false>(C) + slot_bytes<TY, false>(C));
    slot_y = slot_x + slot_bytes<TX, false>(C);
    ask_row(slot_y, yp, C, tid, threads);
    ask_row(slot_x, xp, C, tid, threads);
    asm volatile("cp.async.wait_all;" ::: "memory");
    meet();
    yp = in_slot(slot_y, yp);
    xp = in_slot(slot_x, xp);
  }
  auto all_read = [&] {                            // the slots become r's and h's
    if constexpr (kStage) meet();
  };
  const float inv = 1.f / C;
  const char* gp = reinterpret_cast<const char*>(a.gate);
  if (a.gate && a.rows_per_gate < a.rows)
    gp += (int64_t)((uint64_t)row < (1ull << 32) && a.rows_per_gate < (1ll << 32) ? (uint32_t)row / (uint32_t)a.rows_per_gate
                                                                              : row / a.rows_per_gate) *
          C * (a.wf32 ? 4 : sizeof(TY));
  float2 n[VPT][kP];
  auto normalise = [&](const void* w, const void* bias) {   // n in place
    float mu = 0.f;
    if (a.layer) {
      float2 t = both(0.f);
#pragma unroll
      for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int j = 0; j < kP; ++j) t = add2(t, n[v][j]);
      float s[1] = {t.x + t.y};
      row_sum<1, 8>(s, warps, buf, turn);
      mu = s[0] * inv;
    }
    float2 t = both(0.f);
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        n[v][j] = add2(n[v][j], both(-mu));
        if (a.layer) n[v][j] = mul2(n[v][j], inside<VEC>(v, j, tid, threads, C));
        t = fma2(n[v][j], n[v][j], t);
      }
    float q[1] = {t.x + t.y};
    row_sum<1, 8>(q, warps, buf, turn);
    const float rstd = rsqrtf(q[0] * inv + a.eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int j = 0; j < kP; ++j) n[v][j] = mul2(n[v][j], both(rstd));
      if (w) {
        float2 wv[kP];
        load_w<TY, VEC>(wv, w, a.wf32, v, tid, threads, C);
#pragma unroll
        for (int j = 0; j < kP; ++j) n[v][j] = mul2(n[v][j], wv[j]);
      }
      if (bias) {
        float2 bv[kP];
        load_w<TY, VEC>(bv, bias, a.wf32, v, tid, threads, C);
#pragma unroll
        for (int j = 0; j < kP; ++j) n[v][j] = add2(n[v][j], bv[j]);
      }
    }
  };
  auto join = [&](int v, const float2 (&x)[kP]) {           // n = alpha x + g n
    if (a.gate) {
      float2 g[kP];
      load_w<TY, VEC>(g, gp, a.wf32, v, tid, threads, C);
#pragma unroll
      for (int j = 0; j < kP; ++j) n[v][j] = mul2(n[v][j], g[j]);
    }
#pragma unroll
    for (int j = 0; j < kP; ++j) n[v][j] = fma2(both(a.alpha), x[j], n[v][j]);
    store8<TX, VEC>(kStage ? in_slot(slot_x, rp) : rp, n[v], v, tid, threads, C);
  };
  if constexpr (POST) {
    float2 x[VPT][kP];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      load8<TY, VEC>(n[v], yp, v, tid, threads, C);
      load8<TX, VEC>(x[v], xp, v, tid, threads, C);
    }
    all_read();
    normalise(a.w_post, a.b_post);
#pragma unroll
    for (int v = 0; v < VPT; ++v) join(v, x[v]);
  } else {
    float2 x[VPT][kP];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      load8<TY, VEC>(n[v], yp, v, tid, threads, C);
      load8<TX, VEC>(x[v], xp, v, tid, threads, C);
    }
    all_read();
#pragma unroll
    for (int v = 0; v < VPT; ++v) join(v, x[v]);
  }
  if constexpr (kStage) {
    meet();
    put_row(rp, slot_x, C, tid, threads);
  }
  if (!a.pre) return;
  // h is the norm of r before r's rounding to the stream's type
  normalise(a.w_pre, a.b_pre);
#pragma unroll
  for (int v = 0; v < VPT; ++v) store8<TY, VEC>(kStage ? in_slot(slot_y, hp) : hp, n[v], v, tid, threads, C);
  if constexpr (kStage) {
    meet();
    put_row(hp, slot_y, C, tid, threads);
  }
}

// ---------------------------------------------------------------- backward
// Columns of the partial sums, in this order.
enum { kDwPost, kDbPost, kDwPre, kDbPre, kCols };

// Rows of the stages of the ring: dr, r (stream type), dh, y, one after the other.
template <typename TX, typename TY, bool VEC>
__host__ __device__ inline int stage_bytes(int C) {
  return 2 * slot_bytes<TX, VEC>(C) + 2 * slot_bytes<TY, VEC>(C);
}

// FULL: with means (layer norm) or biases.  RING: rows come through a ring of `stages` rows in
// shared memory, filled by bulk copies that run ahead of the arithmetic without holding registers;
// else (two rows do not fit) each thread reads its columns directly.  Weights lie in shared memory as
// float32; a thread only touches its own columns of them.
//
// Without means every sum of a row is linear in the raw products, the statistics being factors: with
// p = w_post g y and rho, sigma the inverse norms of r and y,
//   sum(dn w_post yhat) = sigma (sum dr p + rho (sum z p - rho^2 mean(z r) sum r p)),
// so six sums and one barrier a row do (32768 rows of 4096: 382 us, with a second sum after the first 456).
// With means the centred rows are summed: three barriers.  More than 512 threads have no registers for the six
// (640 threads, rows of 5120: 495 us against 393 with two sums): two.
template <typename TX, typename TY, bool FULL, bool VEC, bool RING, int MAXT>
__global__ void __launch_bounds__(MAXT) k_norm_bwd(const __grid_constant__ NormArgs a) {
  constexpr bool kOne = !FULL && MAXT <= 512;   // one sum a row
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ alignas(16) float buf[kSumFloats<MAXT <= 512 ? 16 : 32>];
  __shared__ uint64_t full[kMaxStages];
  __shared__ int dead_flag, asked;                          // (asked: rows whose copies have been asked for, where not all)
  volatile int* dead = &dead_flag;
  const int threads = blockDim.x, tid = threadIdx.x, warps = threads >> 5, C = a.C;
  const int64_t first = a.rows * blockIdx.x / gridDim.x, last = a.rows * (blockIdx.x + 1) / gridDim.x;
  int turn = 0;
  const float inv = 1.f / C, inv_mean = a.layer ? inv : 0.f;
  const int stride = threads * kE;                          // floats of one weight
  float* const weights = reinterpret_cast<float*>(dyn);     // w_pre, w_post, gate, and b_post
  uint8_t* const ring = dyn + (FULL ? 4 : 3) * stride * sizeof(float);
  const bool need_y = a.post || a.gate;
  const int bytes_x = slot_bytes<TX, VEC>(C), bytes_y = slot_bytes<TY, VEC>(C);
  auto request = [&](int64_t row) {                         // one thread: the copies of a row
    if (row >= last || (a.lose && row == last - 1)) return;
    const int st = (int)((row - first) % a.stages);
    const uint32_t bar = smem_u32(&full[st]);
    uint8_t* to = ring + (size_t)st * stage_bytes<TX, TY, VEC>(C);
    const void* from[4] = {reinterpret_cast<const TX*>(a.dr) + row * a.dr_row, reinterpret_cast<const TX*>(a.x) + row * a.x_row,
                           reinterpret_cast<const TY*>(a.dh) + row * a.dh_row, reinterpret_cast<const TY*>(a.y) + row * a.y_row};
    const int at[4] = {0, bytes_x, 2 * bytes_x, 2 * bytes_x + bytes_y};
    uint32_t n[4], all = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t bytes = C * (k < 2 ? sizeof(TX) : sizeof(TY));
      n[k] = VEC ? bytes : ((uint32_t)(reinterpret_cast<uintptr_t>(from[k]) & 15) + bytes + 15) & ~15u;
      if (k == 0 || (k == 3 ? need_y : a.pre != 0)) all += n[k];
      else n[k] = 0;
    }
    mbar_expect(bar, all);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n[k])
        bulk_copy(smem_u32(to + at[k]), VEC ? from[k] : reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(from[k]) & ~uintptr_t(15)), n[k],
                  bar);
  };
  clear_sums(buf, kSumFloats<MAXT <= 512 ? 16 : 32>);
  if (RING && tid == 0) {
    dead_flag = 0;
    asked = (int)(last - first) - a.lose;
    for (int i = 0; i < a.stages; ++i) mbar_init(smem_u32(&full[i]), 1);
    fence_async();
  }
  // a thread's eight values as two planes of four, so that neighbouring threads meet different banks
  auto own = [&](int which) { return reinterpret_cast<float4*>(weights + which * stride) + tid; };
  auto keep = [&](int which, const void* p, float none) {   // a weight's columns of this thread to shared memory
    float2 t[kP];
#pragma unroll
    for (int j = 0; j < kP; ++j) t[j] = both(none);
    if (p) load_w<TY, VEC>(t, p, a.wf32, 0, tid, threads, C);
    own(which)[0] = make_float4(t[0].x, t[0].y, t[1].x, t[1].y);
    own(which)[threads] = make_float4(t[2].x, t[2].y, t[3].x, t[3].y);
  };
  auto weight = [&](int which, float2 (&o)[kP]) {
    const float4 x = own(which)[0], y = own(which)[threads];
    o[0] = make_float2(x.x, x.y), o[1] = make_float2(x.z, x.w), o[2] = make_float2(y.x, y.y), o[3] = make_float2(y.z, y.w);
  };
  keep(0, a.w_pre, 1.f);
  keep(1, a.w_post, 1.f);
  if (FULL) keep(3, a.b_post, 0.f);
  __syncthreads();
  if (RING && tid == 0)
    for (int i = 0; i < a.stages; ++i) request(first + i);

  float2 acc[kCols][kP], dg[kP];                            // the biases' columns stay unused without FULL
#pragma unroll
  for (int k = 0; k < kCols; ++k)
#pragma unroll
    for (int j = 0; j < kP; ++j) acc[k][j] = both(0.f);
#pragma unroll
  for (int j = 0; j < kP; ++j) dg[j] = both(0.f);
  const bool cols = VEC ? tid * kE < C : true;              // whether this thread has columns at all
  int64_t group = 0, group_end = a.rows;                    // the gate row at work, and where its rows end
  if (a.gate) {
    group = first / a.rows_per_gate;
    group_end = (group + 1) * a.rows_per_gate;
    keep(2, reinterpret_cast<const char*>(a.gate) + group * C * (a.wf32 ? 4 : sizeof(TY)), 1.f);
  }
  int st = 0, round = 0;
  for (int64_t row = first; row < last; ++row) {
    const uint8_t* at = ring + (size_t)st * stage_bytes<TX, TY, VEC>(C);
    auto fetch = [&](float2 (&o)[kP], int off, auto type, const void* p, int64_t step, bool on) {
      using T = decltype(type);
#pragma unroll
      for (int j = 0; j < kP; ++j) o[j] = both(0.f);
      if (!on) return;
      if constexpr (RING && !VEC) {
        const T* q = reinterpret_cast<const T*>(at + off + (reinterpret_cast<uintptr_t>(reinterpret_cast<const T*>(p) + row * step) & 15));
#pragma unroll
        for (int j = 0; j < kP; ++j) {
          const int c0 = col_of<false>(0, 2 * j, tid, threads), c1 = col_of<false>(0, 2 * j + 1, tid, threads);
          o[j] = make_float2(c0 < C ? ld1(q + c0) : 0.f, c1 < C ? ld1(q + c1) : 0.f);
        }
      } else if constexpr (RING) {
        if (cols) {
          Raw8<T> d;
          const uint4* q = reinterpret_cast<const uint4*>(at + off + tid * kE * (int)sizeof(T));
          *reinterpret_cast<uint4*>(d.v) = q[0];
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(d.v + 4) = q[1];
          widen(o, d);
        }
      } else {
        load8<T, VEC>(o, reinterpret_cast<const T*>(p) + row * step, 0, tid, threads, C);
      }
    };
    if (RING && !mbar_wait(smem_u32(&full[st]), round & 1, dead, a.wait_limit)) {
      if (tid == 0) asked = min(asked, max((int)(row - first) - 1, 0) + a.stages);
    }
    float2 r[kP], dh[kP], y[kP], z[kP], d[kP];
    fetch(r, bytes_x, TX(), a.x, a.x_row, a.pre);
    fetch(dh, 2 * bytes_x, TY(), a.dh, a.dh_row, a.pre);
    fetch(y, 2 * bytes_x + bytes_y, TY(), a.y, a.y_row, need_y);
    fetch(d, 0, TX(), a.dr, a.dr_row, true);
    weight(0, z);
#pragma unroll
    for (int j = 0; j < kP; ++j) z[j] = mul2(dh[j], z[j]);
    // statistics of both rows together
    float mean_z = 0.f;
    if (FULL) {
      float2 t[3] = {both(0.f), both(0.f), both(0.f)};
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        t[0] = add2(t[0], r[j]);
        t[1] = add2(t[1], y[j]);
        t[2] = add2(t[2], z[j]);
      }
      float s[3] = {t[0].x + t[0].y, t[1].x + t[1].y, t[2].x + t[2].y};
      row_sum<3, MAXT <= 512 ? 16 : 32>(s, warps, buf, turn);
      const float mu_r = -s[0] * inv_mean, mu_y = a.post ? -s[1] * inv_mean : 0.f;
      mean_z = s[2] * inv_mean;
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const float2 in = inside<VEC>(0, j, tid, threads, C);
        r[j] = mul2(add2(r[j], both(mu_r)), in);
        y[j] = mul2(add2(y[j], both(mu_y)), in);
      }
    }
    float2 w[kP], g[kP];
    auto gate_weights = [&] {
      if (a.gate && row == group_end) {                      // uniform: the block's rows enter another gate row
        if (!a.gate_direct && cols) {
#pragma unroll
          for (int j = 0; j < kE; ++j) {
            const int c = col_of<VEC>(0, j, tid, threads);
            if (c < C) a.gpart[(blockIdx.x + group) * C + c] = (j & 1) ? dg[j / 2].y : dg[j / 2].x;
          }
        }
#pragma unroll
        for (int j = 0; j < kP; ++j) dg[j] = both(0.f);
        ++group;
        group_end += a.rows_per_gate;
        keep(2, reinterpret_cast<const char*>(a.gate) + group * C * (a.wf32 ? 4 : sizeof(TY)), 1.f);
      }
      weight(1, w);
      if (a.gate) weight(2, g);
    };
    if (kOne) gate_weights();
    constexpr int kQ = kOne ? 6 : 3;
    float2 t[kQ];
#pragma unroll
    for (int k = 0; k < kQ; ++k) t[k] = both(0.f);
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      t[0] = fma2(r[j], r[j], t[0]);
      t[1] = fma2(y[j], y[j], t[1]);
      t[2] = fma2(z[j], r[j], t[2]);
      if constexpr (kOne) {
        float2 p = mul2(w[j], y[j]);
        if (a.gate) p = mul2(g[j], p);
        t[3] = fma2(d[j], p, t[3]);
        t[4] = fma2(z[j], p, t[4]);
        t[5] = fma2(r[j], p, t[5]);
      }
    }
    float q[kQ];
#pragma unroll
    for (int k = 0; k < kQ; ++k) q[k] = t[k].x + t[k].y;
    row_sum<kQ, MAXT <= 512 ? 16 : 32>(q, warps, buf, turn);
    if (RING && tid == 0 && row > first && !*dead) request(row - 1 + a.stages);   // every thread has left the row before
    if (a.pre) {
      const float rstd = rsqrtf(q[0] * inv + a.eps), proj = -q[2] * inv * rstd;   // -mean(z rhat)
      if constexpr (kOne) q[3] += rstd * (q[4] + proj * rstd * q[5]);
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const float2 hat = mul2(r[j], both(rstd));
        acc[kDwPre][j] = fma2(dh[j], hat, acc[kDwPre][j]);
        if (FULL) acc[kDbPre][j] = add2(acc[kDbPre][j], dh[j]);
        const float2 v = fma2(hat, both(proj), FULL ? add2(z[j], both(-mean_z)) : z[j]);
        d[j] = fma2(both(rstd), v, d[j]);
      }
    }
    {
      float2 o[kP];
#pragma unroll
      for (int j = 0; j < kP; ++j) o[j] = mul2(both(a.alpha), d[j]);
      store8<TX, VEC>(reinterpret_cast<TX*>(a.dx) + row * C, o, 0, tid, threads, C);
    }
    const float rstd = a.post ? rsqrtf(q[1] * inv + a.eps) : 1.f;
#pragma unroll
    for (int j = 0; j < kP; ++j) y[j] = mul2(y[j], both(rstd));        // yhat
    if (!kOne) gate_weights();
    if (a.gate) {
      float2 b[kP];
      if (FULL) weight(3, b);
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const float2 n = FULL ? fma2(y[j], w[j], b[j]) : mul2(y[j], w[j]);
        dg[j] = fma2(d[j], n, dg[j]);
        d[j] = mul2(d[j], g[j]);
      }
      if (a.gate_direct) {                         // one row to a gate row: no partials
        if (a.wf32) store8<float, VEC>(reinterpret_cast<float*>(a.dgate) + row * C, dg, 0, tid, threads, C);
        else store8<TY, VEC>(reinterpret_cast<TY*>(a.dgate) + row * C, dg, 0, tid, threads, C);
      }
    }
    if (a.post) {
      float2 u[2] = {both(0.f), both(0.f)};
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        acc[kDwPost][j] = fma2(d[j], y[j], acc[kDwPost][j]);
        if (FULL) acc[kDbPost][j] = add2(acc[kDbPost][j], d[j]);
        d[j] = mul2(d[j], w[j]);
        if constexpr (FULL) u[0] = add2(u[0], d[j]);
        if constexpr (!kOne) u[1] = fma2(d[j], y[j], u[1]);
      }
      float s[FULL ? 2 : 1];
      s[0] = u[1].x + u[1].y;
      if constexpr (FULL) s[1] = u[0].x + u[0].y;
      if constexpr (kOne) s[0] = rstd * q[3];
      else row_sum<FULL ? 2 : 1, MAXT <= 512 ? 16 : 32>(s, warps, buf, turn);
      float mz = 0.f;
      if constexpr (FULL) mz = -s[1] * inv_mean;
      const float proj = -s[0] * inv;
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const float2 v = fma2(y[j], both(proj), FULL ? add2(d[j], both(mz)) : d[j]);
        d[j] = mul2(both(rstd), v);
      }
    }
    store8<TY, VEC>(reinterpret_cast<TY*>(a.dy) + row * C, d, 0, tid, threads, C);
    if (++st == a.stages) {
      st = 0;
      ++round;
    }
  }
#pragma unroll
  for (int j = 0; j < kE; ++j) {
    const int c = col_of<VEC>(0, j, tid, threads);
    if (c >= C) continue;
    if (a.want_cols)
#pragma unroll
      for (int k = 0; k < kCols; ++k)
        a.part[((int64_t)blockIdx.x * kCols + k) * C + c] = (j & 1) ? acc[k][j / 2].y : acc[k][j / 2].x;
    if (a.gate && !a.gate_direct && first < last) a.gpart[(blockIdx.x + group) * C + c] = (j & 1) ? dg[j / 2].y : dg[j / 2].x;
  }
  if constexpr (RING) {
    __syncthreads();
    if (*dead) {                                    // the copies still on their way end before the block does
      int none = 0;
      if (tid == 0) {
        for (int r = max(0, asked - a.stages); r < asked; ++r) mbar_wait(smem_u32(&full[r % a.stages]), (r / a.stages) & 1, &none);
        if (a.status) *a.status = 1;
      }
      __syncthreads();
    }
  }
}

// Adds the partials of every block, in the blocks' order.  blockIdx.y < kCols: a weight's or
// bias's columns; above: gate row blockIdx.y - kCols, over the blocks whose rows meet it.
constexpr int kRedCols = 32, kRedLanes = 8;
struct RedArgs {
  const float *part, *gpart;
  void* out[kCols];
  void* dgate;
  int64_t rows, rows_per_gate;
  int C, blocks, type;   // type: B3R_* of the outputs
};

__device__ __forceinline__ void store_as(void* p, int64_t i, float x, int type) {
  if (type == B3R_F32) reinterpret_cast<float*>(p)[i] = x;
  else if (type == B3R_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
}

__global__ void __launch_bounds__(kRedCols * kRedLanes) k_norm_reduce(const __grid_constant__ RedArgs a, int64_t y0) {
  __shared__ float sh[kRedLanes][kRedCols];
  const int c = blockIdx.x * kRedCols + threadIdx.x;
  const int64_t which = blockIdx.y + y0;
  const float* p;
  int64_t n, stride;
  void* out;
  int64_t at = c;
  if (which < kCols) {
    out = a.out[which];
    p = a.part + which * a.C;
    n = a.blocks;
    stride = (int64_t)kCols * a.C;
  } else {
    const int64_t g = which - kCols, r0 = g * a.rows_per_gate, r1 = r0 + a.rows_per_gate - 1;
    // block b holds rows [rows b / blocks, rows (b + 1) / blocks); the one of row r
    auto owner = [&](int64_t r) {
      int64_t b = r * a.blocks / a.rows;
      while (a.rows * (b + 1) / a.blocks <= r) ++b;
      while (a.rows * b / a.blocks > r) --b;
      return b;
    };
    const int64_t b0 = owner(r0), b1 = owner(r1);
    out = a.dgate;
    p = a.gpart + (b0 + g) * a.C;
    n = b1 - b0 + 1;
    stride = a.C;
    at = g * a.C + c;
  }
  if (!out) return;                                // uniform over the block
  float s = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int64_t i = threadIdx.y; i < n; i += kRedLanes) s += p[i * stride + c];
  }
  sh[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < a.C) {
    float t = 0.f;
#pragma unroll
    for (int l = 0; l < kRedLanes; ++l) t += sh[l][threadIdx.x];
    store_as(out, at, t, a.type);
  }
}

// ---------------------------------------------------------------- launches
constexpr int kMaxC = 8192;

// A kernel's dynamic shared memory limit, raised once on each device to all that its own arrays leave.  (Set to each
// call's need, it could be lowered by another thread's call before the launch that counted on it.)
template <auto F>
int most_smem(const char* what) {
  static uint64_t done = 0;
  int dev;
  B3R_TRY(check_cuda(cudaGetDevice(&dev), what));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (__atomic_load_n(&done, __ATOMIC_RELAXED) & bit)) return B3R_OK;
  cudaFuncAttributes at;
  B3R_TRY(check_cuda(cudaFuncGetAttributes(&at, F), what));
  B3R_TRY(check_cuda(cudaFuncSetAttribute(F, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448 - (int)at.sharedSizeBytes), what));
  __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
  return B3R_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename TX, typename TY, int VPT, bool VEC>
int fwd_kernel(const NormArgs& a, dim3 grid, dim3 block, cudaStream_t s) {
  const int smem = !staged<TY, VEC>() ? 0 : block.y * (slot_bytes<TX, false>(a.C) + slot_bytes<TY, false>(a.C));
  constexpr auto with = k_norm_fwd<TX, TY, VPT, VEC, true>, without = k_norm_fwd<TX, TY, VPT, VEC, false>;
  if (staged<TY, VEC>()) B3R_TRY(a.post ? most_smem<with>("residual_norm") : most_smem<without>("residual_norm"));
  (a.post ? with : without)<<<grid, block, smem, s>>>(a);
  return check_launch("residual_norm");
}

template <typename TX, typename TY, bool VEC>
int fwd_launch(const NormArgs& a, cudaStream_t s) {
  // One warp holds up to 1024 columns (32 a lane); longer rows take up to 8 warps.  Few rows
  // leave the SMs idle either way, so there they are spread over more threads for latency.
  const int C = a.C;
  int threads, vpt;
  if (a.rows >= kSms * 4 && C <= 1024) {
    threads = 32;
    vpt = C <= 256 ? 1 : C <= 512 ? 2 : 4;
  } else {
    threads = std::min(256, std::max(32, (C + kE * 32 - 1) / (kE * 32) * 32));
    vpt = C <= threads * kE ? 1 : C <= threads * kE * 2 ? 2 : 4;
  }
  const dim3 block(threads, threads == 32 ? 4 : 1);
  const int64_t grid = (a.rows + block.y - 1) / block.y;
  B3R_REQUIRE(grid <= 0x7fffffff, "residual_norm: too many rows for one call");
  if (vpt == 1) return fwd_kernel<TX, TY, 1, VEC>(a, (unsigned)grid, block, s);
  if (vpt == 2) return fwd_kernel<TX, TY, 2, VEC>(a, (unsigned)grid, block, s);
  return fwd_kernel<TX, TY, 4, VEC>(a, (unsigned)grid, block, s);
}

int bwd_threads(int C) { return (C + kE * 32 - 1) / (kE * 32) * 32; }

// Blocks of the backward pass: as many as fit the 148 SMs at once (512 threads an SM, by their
// registers), each with a run of rows; of 16 rows at least where that leaves a block for every SM, since
// each block writes partial sums of every column.
int bwd_per_sm(int C) { return std::max(1, std::min(16, 512 / bwd_threads(C))); }
int bwd_blocks(int64_t rows, int C) {
  return (int)std::min<int64_t>({rows, kSms * bwd_per_sm(C), std::max<int64_t>(kSms, rows / 16)});
}

template <typename TX, typename TY, bool FULL, bool VEC, bool RING, int MAXT>
int bwd_kernel(const NormArgs& a, int smem, cudaStream_t s) {
  constexpr auto f = k_norm_bwd<TX, TY, FULL, VEC, RING, MAXT>;
  B3R_TRY(most_smem<f>("residual_norm backward"));
  f<<<bwd_blocks(a.rows, a.C), bwd_threads(a.C), smem, s>>>(a);
  return check_launch("residual_norm backward");
}

template <typename TX, typename TY, bool FULL, bool VEC>
int bwd_launch(NormArgs a, cudaStream_t s) {
  const int threads = bwd_threads(a.C), stage = stage_bytes<TX, TY, VEC>(a.C);
  const int weights = (FULL ? 4 : 3) * threads * kE * 4, room = (227 * 1024) / bwd_per_sm(a.C) - 3 * 1024;   // (static and reserved)
  a.stages = std::min(kMaxStages, (room - weights) / stage);
  if (a.stages >= 2) {
    const int smem = weights + a.stages * stage;
    // registers of a thread: 128, 96 and 64 (18600 bfloat16 rows of 5120 beside a float32 stream with 96: RMS 393 us,
    // layer norm 546; with 64, where they do not hold a row's columns and their sums, 508 and 715)
    if (threads <= 512) return bwd_kernel<TX, TY, FULL, VEC, true, 512>(a, smem, s);
    if (threads <= 640) return bwd_kernel<TX, TY, FULL, VEC, true, 640>(a, smem, s);
    return bwd_kernel<TX, TY, FULL, VEC, true, 1024>(a, smem, s);
  }
  return bwd_kernel<TX, TY, FULL, VEC, false, 1024>(a, weights, s);
}

template <bool FWD, typename TX, typename TY>
int go2(const NormArgs& a, bool vec, cudaStream_t s) {
  if constexpr (FWD) {
    return vec ? fwd_launch<TX, TY, true>(a, s) : fwd_launch<TX, TY, false>(a, s);
  } else {
    const bool full = a.layer || a.biases;
    if (vec) return full ? bwd_launch<TX, TY, true, true>(a, s) : bwd_launch<TX, TY, false, true>(a, s);
    return full ? bwd_launch<TX, TY, true, false>(a, s) : bwd_launch<TX, TY, false, false>(a, s);
  }
}

template <bool FWD>
int go(const NormArgs& a, int stream_type, int dtype, bool vec, cudaStream_t s) {
  if (dtype == B3R_F32) return go2<FWD, float, float>(a, vec, s);
  if (dtype == B3R_BF16)
    return stream_type == B3R_F32 ? go2<FWD, float, __nv_bfloat16>(a, vec, s) : go2<FWD, __nv_bfloat16, __nv_bfloat16>(a, vec, s);
  return stream_type == B3R_F32 ? go2<FWD, float, __half>(a, vec, s) : go2<FWD, __half, __half>(a, vec, s);
}

int common(const b3r_residual_norm* d, NormArgs& a) {
  B3R_REQUIRE(d, "residual_norm: NULL descriptor");
  B3R_REQUIRE(d->dtype == B3R_F32 || d->dtype == B3R_BF16 || d->dtype == B3R_F16, "residual_norm: dtype must be f32, bf16 or f16");
  B3R_REQUIRE(d->stream_dtype == d->dtype || d->stream_dtype == B3R_F32,
              "residual_norm: the residual stream is float32 or of the block's type");
  B3R_REQUIRE(d->weight_dtype == d->dtype || d->weight_dtype == B3R_F32,
              "residual_norm: weights, biases and gates are float32 or of the block's type");
  B3R_REQUIRE(d->rows >= 0 && d->C >= 1 && d->C <= kMaxC, "residual_norm: 1 to %d channels, got %d", kMaxC, d->C);
  B3R_REQUIRE(d->kind == B3R_NORM_LAYER || d->kind == B3R_NORM_RMS, "residual_norm: unknown kind %d", d->kind);
  B3R_REQUIRE(d->eps >= 0.f, "residual_norm: eps must not be negative");
  B3R_REQUIRE(!d->gate || (d->rows_per_gate >= 1 && d->rows % d->rows_per_gate == 0),
              "residual_norm: the rows do not divide into the gate's rows");
  B3R_REQUIRE((d->post || (!d->w_post && !d->b_post)) && (d->pre || (!d->w_pre && !d->b_pre)),
              "residual_norm: weights given for a norm that is switched off");
  a = NormArgs{};
  a.rows = d->rows;
  a.rows_per_gate = d->gate ? d->rows_per_gate : 1;
  a.C = d->C;
  a.layer = d->kind == B3R_NORM_LAYER;
  a.wf32 = d->weight_dtype == B3R_F32;
  a.eps = d->eps;
  a.alpha = d->residual_scale;
  a.w_post = d->w_post;
  a.b_post = d->b_post;
  a.gate = d->gate;
  a.w_pre = d->w_pre;
  a.b_pre = d->b_pre;
  a.post = d->post;
  a.pre = d->pre;
  return B3R_OK;
}

// Whether every row of `p` starts on a vector (16 bytes, 32 of float32; strides: multiples of 8).
bool rows_ok(const void* p, int64_t stride, int type) { return ((uintptr_t)p & (type == B3R_F32 ? 31 : 15)) == 0 && stride % kE == 0; }

bool weights_ok(const NormArgs& a) {
  return aligned16(a.w_post) && aligned16(a.b_post) && aligned16(a.gate) && aligned16(a.w_pre) && aligned16(a.b_pre);
}

int64_t align256(int64_t b) { return (b + 255) & ~int64_t(255); }

}  // namespace
}  // namespace b3r

using namespace b3r;

extern "C" int b3r_residual_norm_fwd(const b3r_residual_norm* d, const void* y, int64_t y_row, const void* x,
                                     int64_t x_row, void* r, void* h, void* stream) {
  NormArgs a;
  B3R_TRY(common(d, a));
  if (a.rows == 0) return B3R_OK;
  B3R_REQUIRE(y && x && r && (h || !a.pre), "residual_norm: NULL tensor");
  a.y = y;
  a.y_row = y_row;
  a.x = x;
  a.x_row = x_row;
  a.r = r;
  a.h = h;
  const int st = d->stream_dtype, dt = d->dtype;
  const bool vec = a.C % kE == 0 && rows_ok(y, y_row, dt) && rows_ok(x, x_row, st) && rows_ok(r, 0, st) && rows_ok(h, 0, dt) && weights_ok(a);
  return go<true>(a, d->stream_dtype, d->dtype, vec, as_stream(stream));
}

extern "C" int64_t b3r_residual_norm_work_bytes(const b3r_residual_norm* d) {
  NormArgs a;
  if (common(d, a) != B3R_OK) return -1;
  if (a.rows == 0) return 0;
  const int64_t blocks = bwd_blocks(a.rows, a.C);
  int64_t n = align256(blocks * kCols * a.C * 4);
  if (a.gate && a.rows_per_gate > 1) n += align256((blocks + a.rows / a.rows_per_gate) * a.C * 4);
  return n;
}

extern "C" int b3r_residual_norm_bwd(const b3r_residual_norm* d, const void* dr, int64_t dr_row, const void* dh,
                                     int64_t dh_row, const void* y, int64_t y_row, const void* r, int64_t r_row,
                                     void* dx, void* dy, void* dgate, void* dw_post, void* db_post, void* dw_pre,
                                     void* db_pre, void* work, void* stream) {
  return b3r_residual_norm_bwd_ex(d, dr, dr_row, dh, dh_row, y, y_row, r, r_row, dx, dy, dgate, dw_post, db_post, dw_pre, db_pre,
                                  work, nullptr, 0, 0, stream);
}

extern "C" int b3r_residual_norm_bwd_ex(const b3r_residual_norm* d, const void* dr, int64_t dr_row, const void* dh,
                                        int64_t dh_row, const void* y, int64_t y_row, const void* r, int64_t r_row,
                                        void* dx, void* dy, void* dgate, void* dw_post, void* db_post, void* dw_pre,
                                        void* db_pre, void* work, int32_t* status, int wait_limit, int flags, void* stream) {
  NormArgs a;
  B3R_TRY(common(d, a));
  B3R_REQUIRE((flags & ~B3R_NORM_TEST_LOST_COPY) == 0, "residual_norm backward: unknown flags");
  a.status = status;
  a.wait_limit = wait_limit > 0 ? wait_limit : kWaitLimit;
  a.lose = flags & B3R_NORM_TEST_LOST_COPY;
  cudaStream_t s = as_stream(stream);
  const int64_t wsz = d->weight_dtype == B3R_F32 ? 4 : 2;
  void* const outs[kCols] = {dw_post, db_post, dw_pre, db_pre};
  if (a.rows == 0) {                               // no rows: the sums are zero
    for (void* o : outs)
      if (o) B3R_TRY(check_cuda(cudaMemsetAsync(o, 0, a.C * wsz, s), "residual_norm backward"));
    return B3R_OK;
  }
  B3R_REQUIRE(dr && dx && dy, "residual_norm backward: NULL tensor");
  B3R_REQUIRE(!a.pre || (dh && r), "residual_norm backward: the norm of r needs dh and r");
  B3R_REQUIRE((!a.post && !a.gate) || y, "residual_norm backward: y is needed");
  B3R_REQUIRE(!a.gate || dgate, "residual_norm backward: dgate is needed");
  B3R_REQUIRE(work && ((uintptr_t)work & 255) == 0, "residual_norm backward: work buffer must be 256-byte aligned");
  B3R_REQUIRE(a.post || (!dw_post && !db_post), "residual_norm backward: no norm of y, so no gradient of its weights");
  B3R_REQUIRE(a.pre || (!dw_pre && !db_pre), "residual_norm backward: no norm of r, so no gradient of its weights");
  a.dr = dr;
  a.dr_row = dr_row;
  a.dh = dh;
  a.dh_row = dh_row;
  a.y = y;
  a.y_row = y_row;
  a.x = r;
  a.x_row = r_row;
  a.dx = dx;
  a.dy = dy;
  a.dgate = dgate;
  const bool need_y = a.post || a.gate;
  a.gate_direct = a.gate && a.rows_per_gate == 1;
  a.biases = a.b_post || db_post || db_pre;
  a.want_cols = dw_post || db_post || dw_pre || db_pre;
  const int blocks = bwd_blocks(a.rows, a.C);
  a.part = reinterpret_cast<float*>(work);
  a.gpart = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + align256((int64_t)blocks * kCols * a.C * 4));
  const int st = d->stream_dtype, dt = d->dtype;
  const bool vec = a.C % kE == 0 && rows_ok(dr, dr_row, st) && rows_ok(dx, 0, st) && rows_ok(dy, 0, dt) &&
                   rows_ok(dgate, 0, d->weight_dtype) && weights_ok(a) &&
                   (!a.pre || (rows_ok(dh, dh_row, dt) && rows_ok(r, r_row, st))) && (!need_y || rows_ok(y, y_row, dt));
  B3R_TRY(go<false>(a, d->stream_dtype, d->dtype, vec, s));
  RedArgs q{};
  q.part = a.part;
  q.gpart = a.gpart;
  for (int k = 0; k < kCols; ++k) q.out[k] = outs[k];
  q.dgate = dgate;
  q.rows = a.rows;
  q.rows_per_gate = a.rows_per_gate;
  q.C = a.C;
  q.blocks = blocks;
  q.type = d->weight_dtype;
  const int64_t y0 = a.want_cols ? 0 : kCols;
  const int64_t y1 = kCols + (a.gate && !a.gate_direct ? a.rows / a.rows_per_gate : 0);
  for (int64_t at = y0; at < y1; at += 65535) {    // gridDim.y's limit
    const dim3 grid((a.C + kRedCols - 1) / kRedCols, (unsigned)std::min<int64_t>(65535, y1 - at));
    k_norm_reduce<<<grid, dim3(kRedCols, kRedLanes), 0, s>>>(q, at);
    B3R_TRY(check_launch("residual_norm column sums"));
  }
  return B3R_OK;
}
