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
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "b3r_status.h"

namespace b3r {
namespace {

constexpr int kE = 8;   // consecutive elements of one vector access

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ld1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void st1(float* p, float x) { *p = x; }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void st1(__half* p, float x) { *p = __float2half_rn(x); }

// Eight elements as they lie in memory (16 or 32 bytes).
template <typename T>
struct alignas(16) Raw8 {
  T v[kE];
};

// The columns of a thread: vector v of VPT holds columns (v * threads + tid) * 8 + j, aligned, or,
// where the row's length or an address does not allow vectors, (v * 8 + j) * threads + tid.
template <bool VEC>
__device__ __forceinline__ int col_of(int v, int j, int tid, int threads) {
  return VEC ? (v * threads + tid) * kE + j : (v * kE + j) * threads + tid;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(Raw8<T>& d, const T* p, int v, int tid, int threads, int C) {
  if constexpr (VEC) {
    const int c = (v * threads + tid) * kE;
    if (c < C) d = *reinterpret_cast<const Raw8<T>*>(p + c);
  } else {
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const int c = col_of<false>(v, j, tid, threads);
      if (c < C) d.v[j] = p[c];
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[kE], int v, int tid, int threads, int C) {
  if constexpr (VEC) {
    const int c = (v * threads + tid) * kE;
    if (c < C) {
      Raw8<T> d;
#pragma unroll
      for (int j = 0; j < kE; ++j) st1(&d.v[j], x[j]);
      *reinterpret_cast<Raw8<T>*>(p + c) = d;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const int c = col_of<false>(v, j, tid, threads);
      if (c < C) st1(p + c, x[j]);
    }
  }
}

// A vector of a weight, bias or gate row, float32 or the activations' type; `none` past the row.
template <typename T, bool VEC>
__device__ __forceinline__ void load_w(float (&o)[kE], const void* p, bool f32, int v, int tid, int threads, int C) {
  if (f32) {
    Raw8<float> d{};
    load8<float, VEC>(d, reinterpret_cast<const float*>(p), v, tid, threads, C);
#pragma unroll
    for (int j = 0; j < kE; ++j) o[j] = d.v[j];
  } else {
    Raw8<T> d{};
    load8<T, VEC>(d, reinterpret_cast<const T*>(p), v, tid, threads, C);
#pragma unroll
    for (int j = 0; j < kE; ++j) o[j] = ld1(&d.v[j]);
  }
}

// Sums of K values over the row's threads (a whole block of `warps` warps, or one warp of a block of
// several rows).  `buf`: 2 x K x 32 floats, used in turn, so one barrier per call is enough.
template <int K>
__device__ __forceinline__ void row_sum(float (&s)[K], int warps, float* buf, int& turn) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], d);
  if (warps == 1) return;
  float* b = buf + turn * 4 * 32;
  turn ^= 1;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) b[k * 32 + w] = s[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float t = lane < warps ? b[k * 32 + lane] : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    s[k] = t;
  }
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
  int post, pre, want_cols, gate_direct;
};

// ---------------------------------------------------------------- forward
template <typename TX, typename TY, int VPT, bool VEC>
__global__ void __launch_bounds__(256) k_norm_fwd(const __grid_constant__ NormArgs a) {
  __shared__ float buf[2 * 4 * 32];
  // blockDim.x threads to a row; blocks of several rows have one warp to a row
  const int threads = blockDim.x, tid = threadIdx.x, warps = threads >> 5, C = a.C;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;                       // uniform over the row's threads
  int turn = 0;
  const TY* yp = reinterpret_cast<const TY*>(a.y) + row * a.y_row;
  const TX* xp = reinterpret_cast<const TX*>(a.x) + row * a.x_row;
  Raw8<TY> yr[VPT];
  Raw8<TX> xr[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    yr[v] = Raw8<TY>{};
    xr[v] = Raw8<TX>{};
    load8<TY, VEC>(yr[v], yp, v, tid, threads, C);
    load8<TX, VEC>(xr[v], xp, v, tid, threads, C);
  }
  const float inv = 1.f / C;
  float n[VPT][kE];
#pragma unroll
  for (int v = 0; v < VPT; ++v)
#pragma unroll
    for (int j = 0; j < kE; ++j) n[v][j] = ld1(&yr[v].v[j]);

  // normalises n in place: columns past C are zero before and are never stored
  auto normalise = [&](const void* w, const void* bias) {
    float mu = 0.f;
    if (a.layer) {
      float s[1] = {0.f};
#pragma unroll
      for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int j = 0; j < kE; ++j) s[0] += n[v][j];
      row_sum<1>(s, warps, buf, turn);
      mu = s[0] * inv;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const float d = n[v][j] - mu;
        if (col_of<VEC>(v, j, tid, threads) < C) q[0] += d * d;
      }
    row_sum<1>(q, warps, buf, turn);
    const float rstd = 1.f / sqrtf(q[0] * inv + a.eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float wv[kE], bv[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j) { wv[j] = 1.f; bv[j] = 0.f; }
      if (w) load_w<TY, VEC>(wv, w, a.wf32, v, tid, threads, C);
      if (bias) load_w<TY, VEC>(bv, bias, a.wf32, v, tid, threads, C);
#pragma unroll
      for (int j = 0; j < kE; ++j) n[v][j] = (n[v][j] - mu) * rstd * wv[j] + bv[j];
    }
  };
  if (a.post) normalise(a.w_post, a.b_post);
  const int64_t grow = a.gate ? row / a.rows_per_gate : 0;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    float g[kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) g[j] = 1.f;
    if (a.gate) {
      const char* gp = reinterpret_cast<const char*>(a.gate) + grow * C * (a.wf32 ? 4 : sizeof(TY));
      load_w<TY, VEC>(g, gp, a.wf32, v, tid, threads, C);
    }
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const float t = a.alpha * ld1(&xr[v].v[j]) + g[j] * n[v][j];
      n[v][j] = col_of<VEC>(v, j, tid, threads) < C ? t : 0.f;
    }
    store8<TX, VEC>(reinterpret_cast<TX*>(a.r) + row * C, n[v], v, tid, threads, C);
  }
  if (!a.pre) return;
  // h is the norm of r before r's rounding to the stream's type
  normalise(a.w_pre, a.b_pre);
#pragma unroll
  for (int v = 0; v < VPT; ++v) store8<TY, VEC>(reinterpret_cast<TY*>(a.h) + row * C, n[v], v, tid, threads, C);
}

// ---------------------------------------------------------------- backward
// Columns of the partial sums, in this order.
enum { kDwPost, kDbPost, kDwPre, kDbPre, kCols };

template <typename TX, typename TY, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) k_norm_bwd(const __grid_constant__ NormArgs a) {
  __shared__ float buf[2 * 4 * 32];
  const int threads = blockDim.x, tid = threadIdx.x, warps = threads >> 5, C = a.C;
  const int64_t first = a.rows * blockIdx.x / gridDim.x, last = a.rows * (blockIdx.x + 1) / gridDim.x;
  const float inv = 1.f / C;
  int turn = 0;
  float acc[kCols][kE], dg[kE];
#pragma unroll
  for (int k = 0; k < kCols; ++k)
#pragma unroll
    for (int j = 0; j < kE; ++j) acc[k][j] = 0.f;
#pragma unroll
  for (int j = 0; j < kE; ++j) dg[j] = 0.f;
  bool in[kE];
#pragma unroll
  for (int j = 0; j < kE; ++j) in[j] = col_of<VEC>(0, j, tid, threads) < C;

  Raw8<TX> drr{}, rr{};
  Raw8<TY> dhr{}, yr{};
  const bool need_y = a.post || a.gate;
  auto fetch = [&](int64_t row) {
    load8<TX, VEC>(drr, reinterpret_cast<const TX*>(a.dr) + row * a.dr_row, 0, tid, threads, C);
    if (a.pre) {
      load8<TX, VEC>(rr, reinterpret_cast<const TX*>(a.x) + row * a.x_row, 0, tid, threads, C);
      load8<TY, VEC>(dhr, reinterpret_cast<const TY*>(a.dh) + row * a.dh_row, 0, tid, threads, C);
    }
    if (need_y) load8<TY, VEC>(yr, reinterpret_cast<const TY*>(a.y) + row * a.y_row, 0, tid, threads, C);
  };
  if (first < last) fetch(first);
  int64_t group = a.gate ? first / a.rows_per_gate : 0;
  for (int64_t row = first; row < last; ++row) {
    float d[kE], r[kE], dh[kE], y[kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      d[j] = ld1(&drr.v[j]);
      r[j] = ld1(&rr.v[j]);
      dh[j] = ld1(&dhr.v[j]);
      y[j] = ld1(&yr.v[j]);
    }
    if (row + 1 < last) fetch(row + 1);            // in flight while this row is worked on
    float z[kE];
    {
      float w[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j) w[j] = 1.f;
      if (a.pre && a.w_pre) load_w<TY, VEC>(w, a.w_pre, a.wf32, 0, tid, threads, C);
#pragma unroll
      for (int j = 0; j < kE; ++j) z[j] = dh[j] * w[j];
    }
    // statistics of both rows together
    float mu_r = 0.f, mu_y = 0.f, mean_z = 0.f;
    if (a.layer) {
      float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kE; ++j) { s[0] += r[j]; s[1] += y[j]; s[2] += z[j]; }
      row_sum<3>(s, warps, buf, turn);
      mu_r = s[0] * inv;
      mu_y = s[1] * inv;
      mean_z = s[2] * inv;
    }
    float q[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      r[j] = in[j] ? r[j] - mu_r : 0.f;
      y[j] = in[j] && a.post ? y[j] - mu_y : y[j];
      q[0] += r[j] * r[j];
      q[1] += y[j] * y[j];
      q[2] += z[j] * r[j];
    }
    row_sum<3>(q, warps, buf, turn);
    if (a.pre) {
      const float rstd = 1.f / sqrtf(q[0] * inv + a.eps), proj = q[2] * inv * rstd;   // mean(z rhat)
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const float hat = r[j] * rstd;
        acc[kDwPre][j] += dh[j] * hat;
        acc[kDbPre][j] += dh[j];
        d[j] += rstd * (z[j] - mean_z - hat * proj);
      }
    }
    {
      float o[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j) o[j] = a.alpha * d[j];
      store8<TX, VEC>(reinterpret_cast<TX*>(a.dx) + row * C, o, 0, tid, threads, C);
    }
    const float rstd = a.post ? 1.f / sqrtf(q[1] * inv + a.eps) : 1.f;
    float w[kE], b[kE], g[kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) { w[j] = 1.f; b[j] = 0.f; g[j] = 1.f; }
    if (a.post && a.w_post) load_w<TY, VEC>(w, a.w_post, a.wf32, 0, tid, threads, C);
    if (a.gate) {
      if (a.post && a.b_post) load_w<TY, VEC>(b, a.b_post, a.wf32, 0, tid, threads, C);
      const int64_t grow = row / a.rows_per_gate;
      if (grow != group) {                         // uniform: the block's rows enter another gate row
        if (!a.gate_direct) {
#pragma unroll
          for (int j = 0; j < kE; ++j)
            if (in[j]) a.gpart[(blockIdx.x + group) * C + col_of<VEC>(0, j, tid, threads)] = dg[j];
        }
#pragma unroll
        for (int j = 0; j < kE; ++j) dg[j] = 0.f;
        group = grow;
      }
      const char* gp = reinterpret_cast<const char*>(a.gate) + grow * C * (a.wf32 ? 4 : sizeof(TY));
      load_w<TY, VEC>(g, gp, a.wf32, 0, tid, threads, C);
#pragma unroll
      for (int j = 0; j < kE; ++j) dg[j] += d[j] * (y[j] * rstd * w[j] + b[j]);
      if (a.gate_direct) {                         // one row to a gate row: no partials
        if (a.wf32) store8<float, VEC>(reinterpret_cast<float*>(a.dgate) + row * C, dg, 0, tid, threads, C);
        else store8<TY, VEC>(reinterpret_cast<TY*>(a.dgate) + row * C, dg, 0, tid, threads, C);
      }
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      d[j] *= g[j];
      if (a.post) {
        y[j] *= rstd;                              // yhat
        acc[kDwPost][j] += d[j] * y[j];
        acc[kDbPost][j] += d[j];
        d[j] *= w[j];
        if (in[j]) { s[0] += d[j]; s[1] += d[j] * y[j]; }
      }
    }
    if (a.post) {
      row_sum<2>(s, warps, buf, turn);
      const float mz = a.layer ? s[0] * inv : 0.f, proj = s[1] * inv;
#pragma unroll
      for (int j = 0; j < kE; ++j) d[j] = rstd * (d[j] - mz - y[j] * proj);
    }
    store8<TY, VEC>(reinterpret_cast<TY*>(a.dy) + row * C, d, 0, tid, threads, C);
  }
#pragma unroll
  for (int j = 0; j < kE; ++j) {
    if (!in[j]) continue;
    const int c = col_of<VEC>(0, j, tid, threads);
    if (a.want_cols)
#pragma unroll
      for (int k = 0; k < kCols; ++k) a.part[((int64_t)blockIdx.x * kCols + k) * C + c] = acc[k][j];
    if (a.gate && !a.gate_direct && first < last) a.gpart[(blockIdx.x + group) * C + c] = dg[j];
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
  if (c < a.C)
    for (int64_t i = threadIdx.y; i < n; i += kRedLanes) s += p[i * stride + c];
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

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename TX, typename TY, bool VEC>
int fwd_launch(const NormArgs& a, cudaStream_t s) {
  // One warp holds up to 1024 columns (32 a lane); longer rows take up to 8 warps.  Few rows
  // leave the SMs idle either way, so there they are spread over more threads for latency.
  const int C = a.C;
  int threads, vpt;
  if (a.rows >= 148 * 4 && C <= 1024) {
    threads = 32;
    vpt = C <= 256 ? 1 : C <= 512 ? 2 : 4;
  } else {
    threads = std::min(256, std::max(32, (C + kE * 32 - 1) / (kE * 32) * 32));
    vpt = C <= threads * kE ? 1 : C <= threads * kE * 2 ? 2 : 4;
  }
  const dim3 block(threads, threads == 32 ? 4 : 1);
  const int64_t grid = (a.rows + block.y - 1) / block.y;
  B3R_REQUIRE(grid <= 0x7fffffff, "residual_norm: too many rows for one call");
  if (vpt == 1) k_norm_fwd<TX, TY, 1, VEC><<<(unsigned)grid, block, 0, s>>>(a);
  else if (vpt == 2) k_norm_fwd<TX, TY, 2, VEC><<<(unsigned)grid, block, 0, s>>>(a);
  else k_norm_fwd<TX, TY, 4, VEC><<<(unsigned)grid, block, 0, s>>>(a);
  return check_launch("residual_norm");
}

int bwd_threads(int C) { return (C + kE * 32 - 1) / (kE * 32) * 32; }

// Blocks of the backward pass: as many as fit the 148 SMs at once, each with a run of rows.
int bwd_blocks(int64_t rows, int C) {
  const int per_sm = std::max(1, std::min(8, 512 / bwd_threads(C)));
  return (int)std::min<int64_t>(rows, 148 * per_sm);
}

template <typename TX, typename TY, bool VEC>
int bwd_launch(const NormArgs& a, cudaStream_t s) {
  const int threads = bwd_threads(a.C), blocks = bwd_blocks(a.rows, a.C);
  if (threads <= 512) k_norm_bwd<TX, TY, VEC, 512><<<blocks, threads, 0, s>>>(a);
  else k_norm_bwd<TX, TY, VEC, 1024><<<blocks, threads, 0, s>>>(a);
  return check_launch("residual_norm backward");
}

template <bool FWD, typename TX, typename TY>
int go2(const NormArgs& a, bool vec, cudaStream_t s) {
  if constexpr (FWD) return vec ? fwd_launch<TX, TY, true>(a, s) : fwd_launch<TX, TY, false>(a, s);
  else return vec ? bwd_launch<TX, TY, true>(a, s) : bwd_launch<TX, TY, false>(a, s);
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

// Whether every row of `p` starts on 16 bytes (strides in elements of 2 or 4 bytes: multiples of 8).
bool rows_ok(const void* p, int64_t stride) { return aligned16(p) && stride % kE == 0; }

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
  const bool vec = a.C % kE == 0 && rows_ok(y, y_row) && rows_ok(x, x_row) && aligned16(r) && aligned16(h) && weights_ok(a);
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
  NormArgs a;
  B3R_TRY(common(d, a));
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
  a.gate_direct = a.gate && a.rows_per_gate == 1;
  a.want_cols = dw_post || db_post || dw_pre || db_pre;
  const int blocks = bwd_blocks(a.rows, a.C);
  a.part = reinterpret_cast<float*>(work);
  a.gpart = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + align256((int64_t)blocks * kCols * a.C * 4));
  const bool vec = a.C % kE == 0 && rows_ok(dr, dr_row) && aligned16(dx) && aligned16(dy) && aligned16(dgate) &&
                   weights_ok(a) && (!a.pre || (rows_ok(dh, dh_row) && rows_ok(r, r_row))) &&
                   ((!a.post && !a.gate) || rows_ok(y, y_row));
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
