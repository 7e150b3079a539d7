// Part 5 of the C ABI: rotary positions.
//
// A section of a head, one per position axis, is `half` pairs (u, w); pair k of the token at
// position p turns by the angle whose cosine and sine the table holds at [p][k]:
//     u' = u c - w s,   w' = w c + u s       (inverse: s -> -s, which is the gradient's map too)
// The pairs lie (k, k + half) apart or side by side (interleaved); elements past the rotated
// part pass through.  Every element is read and written once, so HBM bounds the kernel (and the
// launch, for single tokens).
//
// One thread owns one slot of a token: V pairs, or V elements that pass through, with V the
// widest vector that the layout and the alignment allow.  It reads the slot's cosines and
// sines once and keeps them in registers while it walks over the heads of the queries and of
// the keys, four heads' loads in flight at a time; neighbouring threads own neighbouring slots.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "b3r_status.h"

namespace b3r {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotHeads = 4;   // heads whose loads a thread has in flight

struct RotArgs {
  b3r_rotary_part part[2];
  int64_t tokens, T;             // B * T, and T
  int D, half, axes, heads, lanes, n_pos, slots, rot_slots;
  const float2* table;
  const void* pos;
  int64_t pos_batch, pos_token;
  int pos64, inverse;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// V: elements of one vector.  Half layout: a rotated slot is the vectors at e and e + half.
// Interleaved: a rotated slot is the vector at e, V / 2 pairs (V >= 2).
template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kRotThreads) k_rotary(const __grid_constant__ RotArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  const int slot = (int)(i % a.slots);
  const int64_t rest = i / a.slots;
  const int lane = (int)(rest % a.lanes);
  const int64_t tok = rest / a.lanes;
  if (tok >= a.tokens) return;
  const int64_t b = tok / a.T, t = tok - b * a.T;
  const bool turns = slot < a.rot_slots;
  constexpr int NP = IL ? V / 2 : V;   // pairs of a slot
  float c[NP], s[NP];
  int e;                               // the slot's first element
  if (turns) {
    if constexpr (IL) {
      e = slot * V;
    } else {
      const int per = a.half / V, sec = slot / per;
      e = sec * 2 * a.half + (slot - sec * per) * V;
    }
    int last_ax = -1;
    int64_t p = 0;
    float2 cs[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int el = IL ? e + 2 * j : e + j;
      const int ax = el / (2 * a.half), k = IL ? (el - ax * 2 * a.half) / 2 : el - ax * 2 * a.half;
      if (ax != last_ax) {             // a vector of the interleaved layout may span two sections
        const int64_t at = b * a.pos_batch + t * a.pos_token + ax;
        p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at] : reinterpret_cast<const int32_t*>(a.pos)[at];
        last_ax = ax;
      }
      // a position outside of the table has no angle: its pairs come out as NaN
      const float nan = __int_as_float(0x7fffffff);
      cs[j] = (p >= 0 && p < a.n_pos) ? __ldg(a.table + p * a.half + k) : make_float2(nan, nan);
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      c[j] = cs[j].x;
      s[j] = a.inverse ? -cs[j].y : cs[j].y;
    }
  } else {
    e = a.axes * 2 * a.half + (slot - a.rot_slots) * V;
  }
  using W = Vec<T, V>;
  for (int h0 = lane; h0 < a.heads; h0 += a.lanes * kRotHeads) {
    W lo[kRotHeads], hi[kRotHeads];
    T* to[kRotHeads];
#pragma unroll
    for (int q = 0; q < kRotHeads; ++q) {
      const int h = h0 + q * a.lanes;
      to[q] = nullptr;
      if (h < a.heads) {
        const bool second = h >= a.part[0].heads;
        const b3r_rotary_part& pt = second ? a.part[1] : a.part[0];
        const int hh = second ? h - a.part[0].heads : h;
        const T* from = reinterpret_cast<const T*>(pt.x) + b * pt.x_batch + t * pt.x_token + hh * pt.x_head + e;
        to[q] = reinterpret_cast<T*>(pt.out) + b * pt.out_batch + t * pt.out_token + hh * pt.out_head + e;
        lo[q] = *reinterpret_cast<const W*>(from);
        if (!IL && turns) hi[q] = *reinterpret_cast<const W*>(from + a.half);
      }
    }
#pragma unroll
    for (int q = 0; q < kRotHeads; ++q) {
      if (!to[q]) continue;
      if (turns) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          T& ru = IL ? lo[q].v[2 * j] : lo[q].v[j];
          T& rw = IL ? lo[q].v[(2 * j + 1) % V] : hi[q].v[j];
          const float u = to_f(ru), w = to_f(rw);
          ru = from_f<T>(u * c[j] - w * s[j]);
          rw = from_f<T>(w * c[j] + u * s[j]);
        }
        if (!IL) *reinterpret_cast<W*>(to[q] + a.half) = hi[q];
      }
      *reinterpret_cast<W*>(to[q]) = lo[q];
    }
  }
}

// The widest vector (elements) that every address and section allows: 16 bytes, halved until
// it divides them.
int rot_vector(const RotArgs& a, int n_parts, int esz, bool il) {
  int v = 16 / esz;
  auto fits = [&](int w) {
    const int rot = a.axes * 2 * a.half;
    if (rot % w || a.D % w || (!il && a.half % w)) return false;
    for (int p = 0; p < n_parts; ++p) {
      const b3r_rotary_part& q = a.part[p];
      if (((uintptr_t)q.x | (uintptr_t)q.out) % (w * esz)) return false;
      for (int64_t st : {q.x_batch, q.x_token, q.x_head, q.out_batch, q.out_token, q.out_head})
        if (st % w) return false;
    }
    return true;
  };
  while (v > 1 && !fits(v)) v >>= 1;
  return v;
}

template <typename T, int V, bool IL>
int rot_launch(RotArgs& a, cudaStream_t s) {
  // Heads are spread over `lanes` threads of a slot: one thread walks over kRotHeads heads
  // (their loads in flight at once) unless that would leave the SMs without threads.
  const int64_t per_lane = a.tokens * a.slots;
  int lanes = (a.heads + kRotHeads - 1) / kRotHeads;
  if (per_lane * lanes < (int64_t)148 * 1024) lanes = a.heads;
  a.lanes = lanes;
  const int64_t blocks = (per_lane * lanes + kRotThreads - 1) / kRotThreads;
  B3R_REQUIRE(blocks <= 0x7fffffff, "rotary: too many tokens for one call");
  k_rotary<T, V, IL><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);
  return check_launch("rotary");
}

template <typename T>
int rot_run(RotArgs& a, int n_parts, bool il, bool copy_rest, cudaStream_t s) {
  const int rot = a.axes * 2 * a.half;
  int v = rot_vector(a, n_parts, sizeof(T), il);
  B3R_REQUIRE(!il || v >= 2, "rotary: interleaved pairs must be aligned to a pair (even strides and head size)");
  a.rot_slots = il ? rot / v : rot / 2 / v;
  a.slots = a.rot_slots + (copy_rest ? (a.D - rot) / v : 0);
  if (il) {
    if constexpr (sizeof(T) == 2)
      if (v == 8) return rot_launch<T, 8, true>(a, s);
    return v == 4 ? rot_launch<T, 4, true>(a, s) : rot_launch<T, 2, true>(a, s);
  }
  if constexpr (sizeof(T) == 2)
    if (v == 8) return rot_launch<T, 8, false>(a, s);
  return v == 4 ? rot_launch<T, 4, false>(a, s) : v == 2 ? rot_launch<T, 2, false>(a, s) : rot_launch<T, 1, false>(a, s);
}

}  // namespace
}  // namespace b3r

using namespace b3r;

extern "C" int b3r_rotary(const b3r_rotary_part* parts, int n_parts, int64_t B, int64_t T, int D, int dtype,
                          const float* table, int n_pos, int half, int axes, const void* positions, int pos_is_64,
                          int64_t pos_batch, int64_t pos_token, int interleaved, int inverse, void* stream) {
  B3R_REQUIRE(parts && table, "rotary: NULL argument");
  B3R_REQUIRE(n_parts == 1 || n_parts == 2, "rotary: 1 or 2 parts, got %d", n_parts);
  B3R_REQUIRE(dtype == B3R_F32 || dtype == B3R_BF16 || dtype == B3R_F16, "rotary: dtype must be f32, bf16 or f16");
  B3R_REQUIRE(B >= 0 && T >= 0 && D >= 2 && D <= 1024, "rotary: bad sizes (head size 2..1024)");
  B3R_REQUIRE(axes >= 1 && half >= 1 && (int64_t)axes * 2 * half <= D, "rotary: the rotated part exceeds the head");
  B3R_REQUIRE(n_pos >= 1, "rotary: empty table");
  B3R_REQUIRE(((uintptr_t)table & 7) == 0, "rotary: the table must be 8-byte aligned");
  RotArgs a{};
  bool in_place = true;
  a.heads = 0;
  for (int p = 0; p < n_parts; ++p) {
    B3R_REQUIRE(parts[p].heads >= 0 && (parts[p].heads == 0 || B * T == 0 || (parts[p].x && parts[p].out)),
                "rotary: NULL tensor or negative head count");
    a.part[p] = parts[p];
    a.heads += parts[p].heads;
    const bool same = parts[p].x == parts[p].out && parts[p].x_batch == parts[p].out_batch &&
                      parts[p].x_token == parts[p].out_token && parts[p].x_head == parts[p].out_head;
    in_place = in_place && same;
  }
  if (B == 0 || T == 0 || a.heads == 0) return B3R_OK;
  B3R_REQUIRE(positions, "rotary: NULL positions");
  a.tokens = B * T;
  a.T = T;
  a.D = D;
  a.half = half;
  a.axes = axes;
  a.n_pos = n_pos;
  a.table = reinterpret_cast<const float2*>(table);
  a.pos = positions;
  a.pos64 = pos_is_64;
  a.pos_batch = pos_batch;
  a.pos_token = pos_token;
  a.inverse = inverse;
  cudaStream_t s = as_stream(stream);
  // in place, the elements past the rotated part are where they belong already
  if (dtype == B3R_F32) return rot_run<float>(a, n_parts, interleaved, !in_place, s);
  if (dtype == B3R_BF16) return rot_run<__nv_bfloat16>(a, n_parts, interleaved, !in_place, s);
  return rot_run<__half>(a, n_parts, interleaved, !in_place, s);
}
