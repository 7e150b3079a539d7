// What the attention kernels share: a sequence's place in the tensors, and the argument checks.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "b3r_status.h"

namespace b3r {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Where sequence b lies: its rows' offsets (elements) are batch + row * stride with the rows from
// q0 / k0 on.  Lengths and offsets outside of the tensors are cut to them, so that no index that
// a caller passes leads out of range.
struct AttnSeq {
  int64_t q0, k0;   // first row (packed) or 0
  int ql, kl;
};

__device__ __forceinline__ AttnSeq attn_seq(const b3r_attention_desc& d, int b) {
  AttnSeq s;
  if (d.cu_q) {
    auto cut = [](int64_t x, int64_t hi) { return x < 0 ? int64_t(0) : x > hi ? hi : x; };
    s.q0 = cut(d.cu_q[b], d.Tq);
    s.k0 = cut(d.cu_k[b], d.Tk);
    s.ql = (int)cut(cut(d.cu_q[b + 1], d.Tq) - s.q0, d.Lq);
    s.kl = (int)cut(cut(d.cu_k[b + 1], d.Tk) - s.k0, d.Lk);
  } else {
    s.q0 = s.k0 = 0;
    s.ql = d.q_lens ? min(max(d.q_lens[b], 0), d.Lq) : d.Lq;
    s.kl = d.k_lens ? min(max(d.k_lens[b], 0), d.Lk) : d.Lk;
  }
  return s;
}

// How many keys query i sees: those before the returned bound.
__device__ __forceinline__ int attn_bound(const AttnSeq& s, int i, int causal) {
  return causal ? min(s.kl, max(0, i + 1 + s.kl - s.ql)) : s.kl;
}

template <typename T>
__device__ __forceinline__ T* attn_row(const b3r_attn_tensor& t, int b, int64_t row, int h) {
  return reinterpret_cast<T*>(const_cast<void*>(t.p)) + b * t.batch + row * t.row + h * t.head;
}

__device__ __forceinline__ float f_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float f_of(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T t_of(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 t_of<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half t_of<__half>(float x) { return __float2half_rn(x); }

// A kernel's dynamic shared memory limit, raised once on each device.
template <typename F>
int attn_smem(F* f, uint64_t& done, const char* what) {
  int dev;
  B3R_TRY(check_cuda(cudaGetDevice(&dev), what));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (__atomic_load_n(&done, __ATOMIC_RELAXED) & bit)) return B3R_OK;
  B3R_TRY(check_cuda(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448), what));
  __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
  return B3R_OK;
}

// The argument checks: of the sizes alone, and of everything that a direction reads or writes.
int attn_check_sizes(const b3r_attention_desc* d);
int attn_check(const b3r_attention_desc* d, bool backward);

// Clears the outputs' packed rows that belong to no sequence; before the kernels that write the others.
int attn_clear(const b3r_attention_desc* d, bool backward, cudaStream_t s);

// The tensor map of a (D, rows, heads, batch) tensor in boxes of 64 elements x `box` rows.
int attn_map(CUtensorMap* map, const b3r_attn_tensor& t, int64_t rows, int heads, int batch, int D, int dtype, int box);
// The same tensor as (D, heads, rows, batch), in boxes of 64 elements x G heads x 128 / G rows: row m
// of a box is query m / G, head m % G.
int attn_map_groups(CUtensorMap* map, const b3r_attn_tensor& t, int64_t rows, int heads, int G, int batch, int D, int dtype);

}  // namespace b3r
