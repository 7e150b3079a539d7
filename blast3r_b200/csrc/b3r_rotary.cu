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
// sines once and keeps them in registers while it walks over four heads, the loads
// of two or four in flight at a time; neighbouring threads own neighbouring slots.
//
// Measured on one B200, where a copy moves 6.5 TB/s: 49152 tokens of 2 x 16 float16 heads of 64, half pairs on two
// axes, 78 us (5.2 TB/s); 65536 tokens of 32 + 8 bfloat16 heads of 128, 64 of them turned as interleaved pairs, 293 us
// (4.6 TB/s, at 57 % of the issue slots): latency at 32 warps an SM bounds it; batches of four in
// the half layout (95 us) and 48 warps (86) were slower.  A single token takes 2.9 us.  Sections that no 16-byte
// vector divides take the second kernel.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "b3r_status.h"

namespace b3r {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotHeads = 4;   // heads that a thread walks over

struct RotArgs {
  b3r_rotary_part part[2];
  int64_t T;
  uint32_t threads[2];           // work of each part: tokens * lanes * slots
  int lanes[2];
  int D, half, axes, n_pos, slots, rot_slots;
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
// Interleaved: a rotated slot is the vector at e, V / 2 pairs (V >= 2).  blockIdx.y: the part.
template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kRotThreads, 4) k_rotary(const __grid_constant__ RotArgs a) {
  const int part = blockIdx.y, lanes = a.lanes[part];
  const uint32_t i = blockIdx.x * kRotThreads + threadIdx.x;
  if (i >= a.threads[part]) return;
  const uint32_t rest = i / (uint32_t)a.slots, slot = i - rest * a.slots;
  const uint32_t tok = rest / (uint32_t)lanes, lane = rest - tok * lanes;
  const uint32_t b = tok / (uint32_t)a.T, t = tok - b * (uint32_t)a.T;
  const bool turns = (int)slot < a.rot_slots;
  constexpr int NP = IL ? V / 2 : V;   // pairs of a slot
  constexpr int kRotBatch = IL ? 4 : 2;   // heads whose loads are in flight at once
  float c[NP], s[NP];
  int e;                               // the slot's first element
  if (turns) {
    if constexpr (IL) {
      e = slot * V;
    } else {
      const int per = a.half / V, sec = (int)slot / per;
      e = sec * 2 * a.half + ((int)slot - sec * per) * V;
    }
    // a vector of the half layout lies in one section; one of the interleaved layout may span two
    int ax = e / (2 * a.half), k = e - ax * 2 * a.half;
    if (IL) k /= 2;
    const int64_t at = b * a.pos_batch + t * a.pos_token;
    auto position = [&](int x) -> int64_t {
      return a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at + x] : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[at + x];
    };
    int64_t p = position(ax);
    const float sign = a.inverse ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      if (IL && k == a.half) {
        k = 0;
        p = position(++ax);
      }
      // a position outside of the table has no angle: its pairs come out as NaN
      const float nan = __int_as_float(0x7fffffff);
      const float2 cs = (p >= 0 && p < a.n_pos) ? __ldg(a.table + p * a.half + k) : make_float2(nan, nan);
      c[j] = cs.x;
      s[j] = sign * cs.y;
      ++k;
    }
  } else {
    e = a.axes * 2 * a.half + ((int)slot - a.rot_slots) * V;
  }
  using W = Vec<T, V>;
  const b3r_rotary_part& pt = a.part[part];
  const T* from = reinterpret_cast<const T*>(pt.x) + b * pt.x_batch + t * pt.x_token + lane * pt.x_head + e;
  T* to = reinterpret_cast<T*>(pt.out) + b * pt.out_batch + t * pt.out_token + lane * pt.out_head + e;
  const int64_t from_step = lanes * pt.x_head, to_step = lanes * pt.out_head;
  for (int h = lane; h < pt.heads; h += lanes * kRotBatch) {
    W lo[kRotBatch], hi[kRotBatch];
#pragma unroll
    for (int q = 0; q < kRotBatch; ++q)
      if (h + q * lanes < pt.heads) {
        lo[q] = *reinterpret_cast<const W*>(from + q * from_step);
        if (!IL && turns) hi[q] = *reinterpret_cast<const W*>(from + q * from_step + a.half);
      }
#pragma unroll
    for (int q = 0; q < kRotBatch; ++q) {
      if (h + q * lanes >= pt.heads) break;
      T* o = to + q * to_step;
      if (turns) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          T& ru = IL ? lo[q].v[2 * j] : lo[q].v[j];
          T& rw = IL ? lo[q].v[(2 * j + 1) % V] : hi[q].v[j];
          const float u = to_f(ru), w = to_f(rw);
          ru = from_f<T>(u * c[j] - w * s[j]);
          rw = from_f<T>(w * c[j] + u * s[j]);
        }
        if (!IL) *reinterpret_cast<W*>(o + a.half) = hi[q];
      }
      *reinterpret_cast<W*>(o) = lo[q];
    }
    from += kRotBatch * from_step;
    to += kRotBatch * to_step;
  }
}

// Sections that no 16-byte vector divides.  A block takes `per` whole tokens through shared memory: 16-byte pieces
// of the heads come in with all of a thread's loads in flight, a thread turns one pair of a token in every head
// with its angle in registers, and the pieces go out again.  Measured on one B200 (and with narrower vectors
// straight from memory instead): 214478 tokens of 8 + 4 float16 heads of 120, 51 pairs, 351 us, 3.5 TB/s (777);
// 65536 of 16 + 4 bfloat16 heads of 64, 18 pairs 88 us (189), 20 pairs 89 (124), 20 interleaved 70 (70); 512 of
// these with 19 pairs 4.9 (7.3).  The pairs' two-byte accesses to shared memory bound it.
constexpr int kRowPieces = 6;   // of a thread
constexpr int kRowBytes = kRowPieces * kRotThreads * 16;

// x / d for x d < 2^32: the high half of x ceil(2^32 / d)
struct Div {
  uint32_t d, mul;
  explicit Div(uint32_t n = 1) : d(n), mul(n == 1 ? 0 : (uint32_t)(((uint64_t(1) << 32) + n - 1) / n)) {}
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return mul ? __umulhi(x, mul) : x; }
};
struct RowDivs {
  Div pieces, heads[2], pairs, half;
  int per;
};

template <typename T, bool IL>
__global__ void __launch_bounds__(kRotThreads) k_rotary_rows(const __grid_constant__ RotArgs a, const __grid_constant__ RowDivs v, uint32_t tokens) {
  __shared__ alignas(16) uint4 rows[kRowPieces * kRotThreads];
  const int tid = threadIdx.x;
  const b3r_rotary_part& pt = a.part[blockIdx.y];
  if (pt.heads == 0) return;
  const Div heads = v.heads[blockIdx.y];
  const uint32_t first = blockIdx.x * v.per, n = min(tokens - first, (uint32_t)v.per), all = n * heads.d * v.pieces.d;
  const uint32_t b0 = first / (uint32_t)a.T, t0 = first - b0 * (uint32_t)a.T;
  auto place = [&](uint32_t x, int64_t batch, int64_t token, int64_t head) {   // of piece x, in elements
    const uint32_t row = v.pieces.of(x), i = heads.of(row), h = row - i * heads.d;
    uint32_t t = t0 + i, b = b0;
    if (t >= (uint32_t)a.T) {
      const uint32_t q = t / (uint32_t)a.T;
      b += q;
      t -= q * (uint32_t)a.T;
    }
    return b * batch + t * token + h * head + (x - row * v.pieces.d) * (16 / sizeof(T));
  };
  uint4 x[kRowPieces];
#pragma unroll
  for (int u = 0; u < kRowPieces; ++u)
    if (tid + u * kRotThreads < all)
      x[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(pt.x) +
                                             place(tid + u * kRotThreads, pt.x_batch, pt.x_token, pt.x_head));
#pragma unroll
  for (int u = 0; u < kRowPieces; ++u)
    if (tid + u * kRotThreads < all) rows[tid + u * kRotThreads] = x[u];
  __syncthreads();
  for (uint32_t it = tid; it < n * v.pairs.d; it += kRotThreads) {
    const uint32_t i = v.pairs.of(it), pr = it - i * v.pairs.d, ax = v.half.of(pr), k = pr - ax * v.half.d;
    const uint32_t tok = first + i, b = tok / (uint32_t)a.T;
    const int64_t at = b * a.pos_batch + (tok - b * (uint32_t)a.T) * a.pos_token + ax;
    const int64_t p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at] : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[at];
    const float nan = __int_as_float(0x7fffffff);   // (as in k_rotary)
    const float2 cs = (p >= 0 && p < a.n_pos) ? __ldg(a.table + p * a.half + k) : make_float2(nan, nan);
    const float s = a.inverse ? -cs.y : cs.y;
    T* lo = reinterpret_cast<T*>(rows) + i * heads.d * a.D + ax * 2 * a.half + (IL ? 2 * k : k);
    T* hi = lo + (IL ? 1 : a.half);
#pragma unroll 4
    for (uint32_t h = 0; h < heads.d; ++h, lo += a.D, hi += a.D) {
      const float u = to_f(*lo), w = to_f(*hi);
      *lo = from_f<T>(u * cs.x - w * s);
      *hi = from_f<T>(w * cs.x + u * s);
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kRowPieces; ++u)
    if (tid + u * kRotThreads < all)
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(pt.out) + place(tid + u * kRotThreads, pt.out_batch, pt.out_token, pt.out_head)) =
          rows[tid + u * kRotThreads];
}

// Tensors turned in place: whether two of their elements share memory, or might, where strides are not nested
// or two tensors lie within each other's memory with different batch or token strides.
struct Extent {
  int64_t step, na, nb;   // a dimension's stride in bytes, and its sizes in the two tensors
};
// The largest stride first; apart: from the one's start to the other's; end_a, end_b: bytes of a last piece.
bool rot_meet(const Extent* d, int n, int64_t apart, int64_t end_a, int64_t end_b) {
  if (n == 0) return -end_b < apart && apart < end_a;
  int64_t reach = 0;
  for (int i = 1; i < n; ++i) reach += (std::max(d[i].na, d[i].nb) - 1) * d[i].step;
  if (end_a + end_b + 2 * reach > 8 * d->step) return true;
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t first = std::max(1 - d->na, floor_div(-end_b - reach - apart, d->step));
  const int64_t last = std::min(d->nb - 1, floor_div(end_a + reach - apart, d->step) + 1);
  for (int64_t k = first; k <= last; ++k)
    if (rot_meet(d + 1, n - 1, apart + k * d->step, end_a, end_b)) return true;
  return false;
}
bool rot_overlaps(const b3r_rotary_part* parts, int n_parts, int64_t B, int64_t T, int64_t D, int esz) {
  int64_t step[2][3], size[2][3], begin[2], end[2];
  for (int p = 0; p < n_parts; ++p) {
    const b3r_rotary_part& q = parts[p];
    if (q.heads == 0) return n_parts == 2 && rot_overlaps(parts + 1 - p, 1, B, T, D, esz);
    const int64_t st[3] = {q.x_batch, q.x_token, q.x_head}, n[3] = {B, T, q.heads};
    Extent d[3];
    int dims = 0;
    for (int i = 0; i < 3; ++i) {
      step[p][i] = st[i] * esz;
      size[p][i] = n[i];
      if (n[i] > 1) d[dims++] = Extent{step[p][i], n[i], n[i]};
    }
    std::sort(d, d + dims, [](const Extent& x, const Extent& y) { return x.step < y.step; });
    int64_t reach = D * esz;
    for (int i = 0; i < dims; ++i) {
      if (d[i].step < reach) return true;
      reach += (d[i].na - 1) * d[i].step;
    }
    begin[p] = (int64_t)(uintptr_t)q.x;
    end[p] = begin[p] + reach;
  }
  if (n_parts == 1 || end[0] <= begin[1] || end[1] <= begin[0]) return false;
  int64_t end_a = D * esz, end_b = D * esz;
  Extent d[3];
  int dims = 0;
  for (int i = 0; i < 3; ++i) {
    const int64_t sa = step[0][i], sb = step[1][i], na = size[0][i], nb = size[1][i];
    if (na > 1 && nb > 1 && sa != sb) {
      if (i < 2) return true;
      end_a += (na - 1) * sa;          // heads: a token's as one piece
      end_b += (nb - 1) * sb;
    } else if (na > 1 || nb > 1) {
      d[dims++] = Extent{na > 1 ? sa : sb, na, nb};
    }
  }
  std::sort(d, d + dims, [](const Extent& x, const Extent& y) { return x.step > y.step; });
  return rot_meet(d, dims, begin[1] - begin[0], end_a, end_b);
}

// Whether heads can be moved in 16-byte pieces, and how many tokens fit a block: 0 if none.
template <typename T>
int rot_tokens(const RotArgs& a, int n_parts) {
  int64_t most = 0;
  for (int p = 0; p < n_parts; ++p) {
    const b3r_rotary_part& q = a.part[p];
    const int64_t strides = a.D | q.x_batch | q.x_token | q.x_head | q.out_batch | q.out_token | q.out_head;
    if (strides * (int64_t)sizeof(T) % 16 || ((uintptr_t)q.x | (uintptr_t)q.out) % 16) return 0;
    most = std::max(most, (int64_t)q.heads * a.D * (int64_t)sizeof(T));
  }
  return most == 0 ? 0 : (int)(kRowBytes / most);
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
int rot_launch(RotArgs& a, int n_parts, int64_t tokens, cudaStream_t s) {
  // A slot's heads are spread over threads of kRotHeads each, which share its cosines and sines
  // through registers; where that leaves the SMs without threads, one head to a thread.
  uint32_t most = 0;
  for (int p = 0; p < n_parts; ++p) {
    const int heads = a.part[p].heads;
    int64_t lanes = (heads + kRotHeads - 1) / kRotHeads;
    if (tokens * a.slots * lanes < (int64_t)kSms * 1024) lanes = heads;
    const int64_t n = tokens * a.slots * lanes;
    B3R_REQUIRE(n <= 0x7fffff00, "rotary: too many tokens for one call");
    a.lanes[p] = (int)lanes;
    a.threads[p] = (uint32_t)n;
    most = std::max(most, a.threads[p]);
  }
  k_rotary<T, V, IL><<<dim3((most + kRotThreads - 1) / kRotThreads, n_parts), kRotThreads, 0, s>>>(a);
  return check_launch("rotary");
}

template <typename T>
int rot_run(RotArgs& a, int n_parts, int64_t tokens, bool il, bool copy_rest, cudaStream_t s) {
  const int rot = a.axes * 2 * a.half;
  int v = rot_vector(a, n_parts, sizeof(T), il);
  // (below a block for every SM the slots are spread over more threads: one token 2.5 us against 3.2)
  if (v * (int)sizeof(T) < 16 && tokens >= kSms) {
    if (int per = rot_tokens<T>(a, n_parts)) {
      per = (int)std::max<int64_t>(1, std::min<int64_t>(per, tokens / (kSms * 4)));   // few tokens: spread over the SMs
      const int64_t blocks = (tokens + per - 1) / per;
      B3R_REQUIRE(tokens <= 0x7fffffff, "rotary: too many tokens for one call");
      RowDivs dv;
      dv.pieces = Div(a.D * sizeof(T) / 16);
      for (int p = 0; p < n_parts; ++p) dv.heads[p] = Div(std::max(1, a.part[p].heads));
      dv.pairs = Div(a.axes * a.half);
      dv.half = Div(a.half);
      dv.per = per;
      const dim3 grid((unsigned)blocks, n_parts);
      if (il) k_rotary_rows<T, true><<<grid, kRotThreads, 0, s>>>(a, dv, (uint32_t)tokens);
      else k_rotary_rows<T, false><<<grid, kRotThreads, 0, s>>>(a, dv, (uint32_t)tokens);
      return check_launch("rotary");
    }
  }
  B3R_REQUIRE(!il || v >= 2, "rotary: interleaved pairs must be aligned to a pair (even strides and head size)");
  a.rot_slots = il ? rot / v : rot / 2 / v;
  a.slots = a.rot_slots + (copy_rest ? (a.D - rot) / v : 0);
  if (il) {
    if constexpr (sizeof(T) == 2)
      if (v == 8) return rot_launch<T, 8, true>(a, n_parts, tokens, s);
    return v == 4 ? rot_launch<T, 4, true>(a, n_parts, tokens, s) : rot_launch<T, 2, true>(a, n_parts, tokens, s);
  }
  if constexpr (sizeof(T) == 2)
    if (v == 8) return rot_launch<T, 8, false>(a, n_parts, tokens, s);
  return v == 4 ? rot_launch<T, 4, false>(a, n_parts, tokens, s) : v == 2 ? rot_launch<T, 2, false>(a, n_parts, tokens, s) : rot_launch<T, 1, false>(a, n_parts, tokens, s);
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
  B3R_REQUIRE(B >= 0 && T >= 0 && T <= 0x7fffffff && D >= 2 && D <= 1024, "rotary: bad sizes (head size 2..1024)");
  B3R_REQUIRE(axes >= 1 && half >= 1 && (int64_t)axes * 2 * half <= D, "rotary: the rotated part exceeds the head");
  B3R_REQUIRE(n_pos >= 1, "rotary: empty table");
  B3R_REQUIRE(((uintptr_t)table & 7) == 0, "rotary: the table must be 8-byte aligned");
  RotArgs a{};
  bool in_place = true;
  int64_t heads = 0;
  for (int p = 0; p < n_parts; ++p) {
    B3R_REQUIRE(parts[p].heads >= 0 && (parts[p].heads == 0 || B * T == 0 || (parts[p].x && parts[p].out)),
                "rotary: NULL tensor or negative head count");
    a.part[p] = parts[p];
    heads += parts[p].heads;
    const bool same = parts[p].x == parts[p].out && parts[p].x_batch == parts[p].out_batch &&
                      parts[p].x_token == parts[p].out_token && parts[p].x_head == parts[p].out_head;
    in_place = in_place && same;
  }
  if (B == 0 || T == 0 || heads == 0) return B3R_OK;
  if (in_place)
    B3R_REQUIRE(!rot_overlaps(parts, n_parts, B, T, D, dtype == B3R_F32 ? 4 : 2),
                "rotary in place: elements of the tensors overlap in memory, or might; turn copies of them");
  B3R_REQUIRE(positions, "rotary: NULL positions");
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
  if (dtype == B3R_F32) return rot_run<float>(a, n_parts, B * T, interleaved, !in_place, s);
  if (dtype == B3R_BF16) return rot_run<__nv_bfloat16>(a, n_parts, B * T, interleaved, !in_place, s);
  return rot_run<__half>(a, n_parts, B * T, interleaved, !in_place, s);
}
