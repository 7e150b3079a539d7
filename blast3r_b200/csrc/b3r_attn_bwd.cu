// Attention's backward pass on the 5th-generation tensor cores, with P = exp(S - lse) recomputed:
//   delta = do . o,  dv = P^T do,  dP = do v^T,  dS = P (dP - delta),  dq = scale dS k,  dk = scale dS^T q
//
// Two kernels, so that every sum has one owner and a fixed order (no atomics):
//   k_attn_dq    a block owns 128 rows (queries x heads of a group) and walks over the keys; it
//                computes delta on the way in and leaves it for the other kernel
//   k_attn_dkv   a block owns 128 keys and walks over the queries of every head that shares them,
//                with S^T = K Q^T and dP^T = V dO^T, so that P^T and dS^T have the keys' rows
// In both, warp 8 loads tiles by TMA into a ring, warp 9 issues the products, and two warpgroups
// do the elementwise part, one row and half of the columns to a thread.  P and dS go back to
// tensor memory as 16-bit pairs and are read there as the left operands of the products that
// follow; they are rounded to the operands' type for it.  S, dP, delta and the sums are float32.
//
// Splitting the pass in two computes S and dP twice (7 products instead of 5); the
// alternative adds dq to memory from every key block, which needs atomics or an order to wait for.
#include <algorithm>
#include <type_traits>
#include "b3r_attn.cuh"
#include "b3r_tc.cuh"

namespace b3r {
namespace {

constexpr int kThreads = 384;
constexpr int kMaxStages = 4;   // of each ring
// an elementwise thread holds 64 columns of P and of dP: registers move over from the third warpgroup
// (256 x 208 + 128 x 88 = 384 x 168, what the block was launched with)
__device__ __forceinline__ void few_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }
__device__ __forceinline__ void many_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }

// P^T is rounded to the operands' type for dv.  In float16 the small probabilities of long rows
// would be subnormal, so P is carried 2^11 times as large (P <= 1); the factor is taken out of dS in
// float32 and of dv at the end, both exactly.
template <typename T>
constexpr float kLogScaleP = __is_same(T, __half) ? 11.f : 0.f;
template <typename T>
constexpr float kScaleP = __is_same(T, __half) ? 2048.f : 1.f;

// In float16 dS is carried 2^k times as large too, with the largest k that cannot overflow: |dS| is at most
// 2 |do_i| |v_j|, since o is a mean of rows of v.  Gradients of any size then keep their 11 bits.
template <typename T>
__device__ __forceinline__ float scale_ds(const float2* range, int head) {
  if constexpr (!__is_same(T, __half)) return 1.f;
  const float2 r = range[head];
  const float most = 2.f * sqrtf(r.x) * sqrtf(r.y);
  if (!(most > 0.f) || isinf(most)) return 1.f;
  return exp2f(fminf(fmaxf(floorf(log2f(32768.f / most)), -24.f), 24.f));
}

// What is added to a query's raw scores, so that scale times them is the logarithm of P (as it is carried).
template <typename T>
__device__ __forceinline__ float shift_of(float lse, float scale) { return (kLogScaleP<T> / kLog2e - lse) / scale; }

struct alignas(64) BwdArgs {
  CUtensorMap q, go, k, v;    // boxes of 128 rows of a head
  CUtensorMap qg, gog, og;    // boxes of whole groups, where q_tma
  b3r_attention_desc d;
  int q_tiles, k_tiles;       // row tiles of a key/value head's queries, and key tiles, of the longest sequence
  int q_splits, k_splits;     // blocks along the keys for dq, along the queries for dk and dv
  int dq_k_stages, dq_v_stages;    // rings of K and V in k_attn_dq
  int q_stages, go_stages, group;  // rings of Q and dO in k_attn_dkv
  int q_tma;                       // the heads of a group divide 128
  int G;
  int lose;                   // a test: the first block of each kernel never gets its first tile
  float* delta;               // [B][Hq][Lq]
  float2* range;              // float16: [B][Hkv], the largest |do|^2 and |v|^2 of a row;
  int* far;                   // and [B][Hkv], whether lse / scale or delta of a row is above kMostInParts
  float* part_q;              // [q_splits][B Hkv][rows][D]
  float* part_k;              // [k_splits][2][B Hkv][Lk][D]: dk, dv
};

constexpr int kStepBytes = kTileRows * 32;
// A float as 2^8 a + b + 2^-8 c + 2^-14 d with a .. d of the operands' type: to 24 bits at least, in
// float16 for magnitudes from 1e-6 to 1.6e7 (its own numbers end at 6e4, and are coarse below 6e-5).
__host__ __device__ constexpr float weight_of(int k) { return k == 0 ? 256.f : k == 1 ? 1.f : k == 2 ? 1.f / 256.f : 1.f / 16384.f; }
// Up to 256 * 65504 the parts are float16 numbers.  lse / scale is about the largest raw score, and delta a sum of D
// products, so both can lie above.  k_attn_dq, which meets every row, marks the heads where one does; there the
// threads that read S^T and dP^T subtract in float32.  (bfloat16 has float32's range.)
constexpr float kMostInParts = 1.6e7f;
constexpr int kPlain = 4;   // stages of those, three of them needed: t + 2 may be written while tile t is at work

struct Shared {
  uint64_t fix, own_full, full[2][kMaxStages], empty[2][kMaxStages], s_full[2], s_read, dp_full, p_full, ds_full, done, own_ready;
  uint64_t st_full[kPlain], st_empty[2];
  uint32_t tmem;
  int dead;
  float delta[kTileRows];
  alignas(16) float plain[kPlain][2][kTileRows];      // k_attn_dkv, far statistics: what is added to S^T and to dP^T
  // k_attn_dkv: one more step of 16 for S^T and dP^T, which subtracts each query's lse and delta in the tensor
  // cores: the weights below times (per stage and product) four numbers of the operands' type each
  alignas(128) uint4 weights[kStepBytes / 16], stat[2][2][kStepBytes / 16];
};

// Which head and tile a block works on: heads in groups whose tensors fit L2; `heavy_first`
// says on which side of a causal triangle the long tiles lie.
__device__ __forceinline__ void place(int id, int tiles, int group, int heads, bool last_first, int& head, int& tile) {
  const int gsz = group * tiles, g = id / gsz, r = id - g * gsz, width = min(group, heads - g * group);
  head = g * group + r % width;
  tile = last_first ? tiles - 1 - r / width : r / width;
}

__device__ __forceinline__ void init_shared(Shared& sh) {
  mbar_init(smem_u32(&sh.fix), 1);
  mbar_init(smem_u32(&sh.own_full), 1);
  mbar_init(smem_u32(&sh.own_ready), 8);
  for (int i = 0; i < kMaxStages; ++i)
    for (int k = 0; k < 2; ++k) {
      mbar_init(smem_u32(&sh.full[k][i]), 1);
      mbar_init(smem_u32(&sh.empty[k][i]), 1);
    }
  for (int i = 0; i < kPlain; ++i) mbar_init(smem_u32(&sh.st_full[i]), 1);
  for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sh.st_empty[i]), 1);
  mbar_init(smem_u32(&sh.s_full[0]), 1);
  mbar_init(smem_u32(&sh.s_full[1]), 1);
  mbar_init(smem_u32(&sh.s_read), 8);
  mbar_init(smem_u32(&sh.dp_full), 1);
  mbar_init(smem_u32(&sh.p_full), 8);
  mbar_init(smem_u32(&sh.ds_full), 8);
  mbar_init(smem_u32(&sh.done), 1);
  sh.dead = 0;
  fence_async();
}

__device__ __forceinline__ void finish(Shared& sh, int32_t* status, int warp, bool used) {
  tc_fence_before();
  __syncthreads();
  if (*(volatile int*)&sh.dead) {                      // copies that a failed wait left behind
    for (int t = 0; t < 100; ++t) __nanosleep(1000);
    if (threadIdx.x == 0 && status) *status = 1;
    __syncthreads();
  }
  if (warp == 9 && used) {
    tc_fence_after();
    tc_free(sh.tmem, 512);
  }
}

// A warp's 32 rows of 32 columns of an accumulator, times f: to rows of 16-bit values through the warp's
// 2 KB of shared memory (four lanes write the 64 bytes of a row; chunk c of row x lies at c ^ (x / 2 % 4)),
// or to rows of float32 parts.  `row`: whether this thread's row is written at all.
template <typename T>
__device__ __forceinline__ void write32(uint32_t tmem, bool has, float f, T* out, float* part, int D, int c0, bool row, uint8_t* box_) {
  const int lane = threadIdx.x & 31;
  uint32_t o[32];
  float v[32];
  if (has) {
    tc_ld32(tmem, o);
    tc_wait_ld(o);
  }
#pragma unroll
  for (int e = 0; e < 32; ++e) v[e] = has ? __uint_as_float(o[e]) * f : 0.f;
  if (part) {
    if (row)
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        if (c0 + e < D) *reinterpret_cast<float4*>(part + c0 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    return;
  }
  uint4* const box = reinterpret_cast<uint4*>(box_);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 4; ++e)
    box[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_uint4(pack2(v[8 * e], v[8 * e + 1], T()), pack2(v[8 * e + 2], v[8 * e + 3], T()),
                                                         pack2(v[8 * e + 4], v[8 * e + 5], T()), pack2(v[8 * e + 6], v[8 * e + 7], T()));
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 32; x += 8) {
    const int y = x + (lane >> 2), c = lane & 3;
    T* const to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, row ? reinterpret_cast<uint64_t>(out) : 0, y));
    const uint4 z = box[y * 4 + (c ^ ((y >> 1) & 3))];
    if (to && c0 + c * 8 < D) *reinterpret_cast<uint4*>(to + c0 + c * 8) = z;
  }
}

// The largest |do|^2 and |v|^2 of a row among the heads that share keys and values.  A block takes 1024
// rows of one head; the maximum of non-negative floats is that of their bits, in any order.  One pass over do and v.
constexpr int kRangeRows = 1024;
template <typename T>
__global__ void __launch_bounds__(256) k_attn_range(const __grid_constant__ BwdArgs a, int chunks) {
  __shared__ float part[8];
  const b3r_attention_desc& d = a.d;
  const int b = blockIdx.x / chunks, first = (blockIdx.x - b * chunks) * kRangeRows;
  const bool of_v = (int)blockIdx.y >= d.Hq;
  const int h = of_v ? blockIdx.y - d.Hq : blockIdx.y, kv = of_v ? h : h / a.G;
  const AttnSeq s = attn_seq(d, b);
  const int last = min(first + kRangeRows, of_v ? s.kl : s.ql);
  float most = 0.f;
  for (int i = first + threadIdx.x; i < last; i += 256) {
    const uint4* x = reinterpret_cast<const uint4*>(attn_row<const T>(of_v ? d.v : d.d_o, b, (of_v ? s.k0 : s.q0) + i, h));
    float2 sum = make_float2(0.f, 0.f);
    for (int c = 0; c < d.D / 8; ++c) {
      const uint4 u = x[c];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = unpack2(w[e], T());
        sum = __ffma2_rn(y, y, sum);
      }
    }
    most = fmaxf(most, sum.x + sum.y);                 // (a NaN is passed over: it has no size)
  }
#pragma unroll
  for (int t = 16; t > 0; t >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, t));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) most = fmaxf(most, part[i]);
    float2* r = a.range + (int64_t)b * d.Hkv + kv;
    atomicMax(reinterpret_cast<int*>(of_v ? &r->y : &r->x), __float_as_int(most));
  }
}

// ---------------------------------------------------------------- dq
// Tensor memory: S at 0, dP at 128, dq at 256, and the block's own rows of Q and dO after it, as left operands.
// The next S starts as soon as this one has been read; dS overwrites dP, each half in place.  A left operand in
// shared memory costs about 100 cycles for each 16 of the head size where one in tensor memory costs the product's 64,
// so Q and dO are copied over once.  Measured on one B200: 2 x 4096 causal, 32/8 heads of 128, 353 us (1168 TFLOP/s over
// the three products: tensor pipe 59 % busy, the elementwise part beside it); 20 packed sequences of up to 1025,
// 16 heads of 64, 134 us (a third of a block's time is its start and end).
template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 1) k_attn_dq(const __grid_constant__ BwdArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  constexpr int kBlocks = DP / 64, kTile = kBlocks * kBlockBytes, kQ = 256 + DP, kGo = kQ + DP / 2;
  constexpr bool kBf = __is_same(T, __nv_bfloat16);
  Shared& sh = *reinterpret_cast<Shared*>(base + (a.dq_k_stages + a.dq_v_stages) * kTile);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
  const b3r_attention_desc& d = a.d;
  const int G = a.G, split = blockIdx.x % a.q_splits;
  int head, tile;
  place(blockIdx.x / a.q_splits, a.q_tiles, a.group, d.B * d.Hkv, true, head, tile);
  const int b = head / d.Hkv, kv = head % d.Hkv;
  const AttnSeq s = attn_seq(d, b);
  const int rows = (d.cu_q ? s.ql : d.Lq) * G, m0 = tile * kTileRows;
  if (m0 >= rows) return;
  int n = 0, first = 0;
  {
    const int last = min(m0 + kTileRows, s.ql * G) - 1;
    const int all = last < m0 ? 0 : (attn_bound(s, last / G, d.causal) + kTileRows - 1) / kTileRows;
    const int per = (all + a.q_splits - 1) / a.q_splits;
    first = split * per;
    n = min(max(all - first, 0), per);
  }
  if (threadIdx.x == 0) init_shared(sh);
  if (warp == 9 && n > 0) tc_alloc(smem_u32(&sh.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  volatile int* dead = &sh.dead;
  const int steps = (d.D + 15) / 16;
  Ring kr{smem_u32(base), base, sh.full[0], sh.empty[0], a.dq_k_stages};
  Ring vr{smem_u32(base) + a.dq_k_stages * kTile, base + a.dq_k_stages * kTile, sh.full[1], sh.empty[1], a.dq_v_stages};
  // the block's own rows pass through stages that the rings reach last: Q and O through K's, dO through V's
  const int at_q = (a.dq_k_stages - 1) * kTile, at_o = (a.dq_k_stages - 2) * kTile, at_go = (a.dq_k_stages + a.dq_v_stages - 1) * kTile;

  if (warp >= 8) {
    few_registers();
    if (warp == 8 && n > 0) {
      int fixes = 0;
      const int batch = d.cu_k ? 0 : b;
      if (a.q_tma && lane == 0) {      // rows past the end only reach their own row of dq
        const uint32_t bar = smem_u32(&sh.own_full);
        const int row = (int)s.q0 + m0 / G, bq = d.cu_q ? 0 : b;
        mbar_expect(bar, 3 * kTile);
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) {
          tma_box(kr.data + at_q + c * kBlockBytes, &a.qg, c * 64, kv * G, row, bq, bar);
          tma_box(kr.data + at_go + c * kBlockBytes, &a.gog, c * 64, kv * G, row, bq, bar);
          tma_box(kr.data + at_o + c * kBlockBytes, &a.og, c * 64, kv * G, row, bq, bar);
        }
      }
      const int free_until = min(a.dq_k_stages - 2, a.dq_v_stages - 1);
      for (int it = 0; it < n; ++it) {
        const int t = (first + it) * kTileRows;
        if (it == free_until) mbar_wait(smem_u32(&sh.own_ready), 0, dead);
        // dS is zero past the last key and meets K's rows there, so they are cleared
        if (a.lose && blockIdx.x + it == 0) kr.step();   // (a test: it never comes)
        else ring_load<kBlocks, kTileRows>(kr, &a.k, (int)s.k0 + t, kv, batch, s.kl - t, true, &sh.fix, fixes, lane, dead);
        ring_load<kBlocks, kTileRows>(vr, &a.v, (int)s.k0 + t, kv, batch, s.kl - t, false, &sh.fix, fixes, lane, dead);
      }
    } else if (warp == 9 && n > 0) {
      const uint32_t on = elect_one();
      const uint32_t id_s = mma_idesc(kBf, 128, 128, false), id_o = mma_idesc(kBf, 128, (d.D + 15) & ~15, true);
      int k_now = 0, k_next = 0, sv = 0, last_round = 0;
      auto scores = [&]() {                            // S = Q K^T
        k_next = kr.next(dead);
        tc_fence_after();
        tile_product_ts<kBlocks, kTileRows>(tmem, tmem + kQ, kr.data + k_next * kTile, id_s, steps, on);
        tc_commit(smem_u32(&sh.s_full[0]), on);
      };
      auto grads = [&]() {                             // dP = dO V^T
        last_round = vr.round;
        sv = vr.next(dead);
        tc_fence_after();
        tile_product_ts<kBlocks, kTileRows>(tmem + 128, tmem + kGo, vr.data + sv * kTile, id_s, steps, on);
        tc_commit(smem_u32(&sh.dp_full), on);
        tc_commit(smem_u32(&sh.empty[1][sv]), on);
      };
      mbar_wait(smem_u32(&sh.own_ready), 0, dead);
      scores();
      grads();
      for (int it = 0; it < n; ++it) {
        k_now = k_next;
        if (it + 1 < n) {
          mbar_wait(smem_u32(&sh.s_read), it & 1, dead);
          scores();
        }
        mbar_wait(smem_u32(&sh.ds_full), it & 1, dead);
        tc_fence_after();
        tile_gather<kTileRows>(tmem + 256, tmem + 128, 64, kr.data + k_now * kTile, id_o, it > 0, on);   // dq += dS K
        tc_commit(smem_u32(&sh.empty[0][k_now]), on);
        if (it + 1 < n) grads();
      }
      tc_commit(smem_u32(&sh.done), on);
      mbar_wait(smem_u32(&sh.empty[1][sv]), last_round & 1, dead);   // no arrival is left behind
      mbar_wait(smem_u32(&sh.done), 0, dead);
    }
  } else {
    many_registers();
    const int w = warp >> 2, r = threadIdx.x & 127, m = m0 + r;
    const int i = m / G, h = kv * G + m - i * G;
    const bool row = m < rows, live = row && i < s.ql;
    const int bound = live ? attn_bound(s, i, d.causal) : 0;
    const uint32_t quarter = tmem + ((uint32_t)(warp & 3) << 21);
    const float c = d.scale * kLog2e;
    const float lse_in = bound > 0 ? *attn_row<const float>(d.lse, b, s.q0 + i, h) : 0.f;
    // one group brings the rows of Q into tensor memory, the other those of dO and, with O, delta
    {
      uint4 x[DP / 8], y[DP / 8];
      if (a.q_tma && n > 0) {
        mbar_wait(smem_u32(&sh.own_full), 0, dead);
        const uint8_t* mine = base + (w ? at_go : at_q) + r * 128;
        const uint8_t* out = base + at_o + r * 128;
#pragma unroll
        for (int cb = 0; cb < DP / 8; ++cb) {
          const int at = (cb >> 3) * kBlockBytes + (((cb & 7) ^ (r & 7)) << 4);
          x[cb] = *reinterpret_cast<const uint4*>(mine + at);
          if (w) y[cb] = *reinterpret_cast<const uint4*>(out + at);
        }
      } else {
        const int64_t qr = s.q0 + (live ? i : 0);
        const int qh = live ? h : kv * G;
        const uint4* mine = reinterpret_cast<const uint4*>(attn_row<const T>(w ? d.d_o : d.q, b, qr, qh));
        const uint4* out = reinterpret_cast<const uint4*>(attn_row<const T>(d.o, b, qr, qh));
#pragma unroll
        for (int cb = 0; cb < DP / 8; ++cb) {
          const bool in = live && cb * 8 < d.D;
          x[cb] = in ? mine[cb] : make_uint4(0, 0, 0, 0);
          y[cb] = in && w ? out[cb] : make_uint4(0, 0, 0, 0);
        }
      }
      if (w) {
        float2 dot[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int cb = 0; cb < DP / 8; ++cb) {
          const uint32_t* xe = reinterpret_cast<const uint32_t*>(&x[cb]);
          const uint32_t* ye = reinterpret_cast<const uint32_t*>(&y[cb]);
#pragma unroll
          for (int e = 0; e < 4; ++e) dot[e & 1] = __ffma2_rn(unpack2(xe[e], T()), unpack2(ye[e], T()), dot[e & 1]);
        }
        const float delta = (dot[0].x + dot[0].y) + (dot[1].x + dot[1].y);
        sh.delta[r] = delta;
        if (live && split == 0) a.delta[((int64_t)b * d.Hq + h) * d.Lq + i] = delta;
        if (!kBf && bound > 0 && split == 0 && !(fmaxf(fabsf(shift_of<T>(lse_in, d.scale)), fabsf(delta)) <= kMostInParts))
          atomicExch(a.far + head, 1);
      }
      if (n > 0) {
#pragma unroll
        for (int cb = 0; cb < DP / 8; cb += 8)
          tc_st32(quarter + (w ? kGo : kQ) + cb * 4, reinterpret_cast<const uint32_t*>(x) + cb * 4);
        tc_wait_st();
        fence_async();                                 // the stages may be loaded again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.own_ready));
      }
      bar_sync(1, 256);
    }
    const float delta = sh.delta[r], lse = lse_in == -INFINITY ? INFINITY : lse_in * kLog2e;   // nothing seen: P = 0
    const float up = scale_ds<T>(a.range, head);
    const float2 cc = make_float2(c, c), ll = make_float2(-lse, -lse), dd = make_float2(-delta * up, -delta * up), uu = make_float2(up, up);
    const int sees = row ? bound : s.kl;               // past the rows nothing is written, so no mask is needed there
    for (int it = 0; it < n; ++it) {
      const int lim = sees - (first + it) * kTileRows - w * 64;      // of this thread's 64 keys, how many its row sees
      const uint32_t at = quarter + w * 64;
      mbar_wait(smem_u32(&sh.s_full[0]), it & 1, dead);
      tc_fence_after();
      uint32_t p[64], g[64];
      tc_ld32(at, p);
      tc_ld32(at + 32, p + 32);
      tc_wait_ld(p);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.s_read));
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])), cc, ll);
        p[e] = __float_as_uint(ex2(x.x));
        p[e + 1] = __float_as_uint(ex2(x.y));
      }
      mbar_wait(smem_u32(&sh.dp_full), it & 1, dead);
      tc_fence_after();
      tc_ld32(at + 128, g);
      tc_ld32(at + 160, g + 32);
      tc_wait_ld(g);
      const bool whole = __all_sync(0xffffffffu, lim >= 64);
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        float2 x = make_float2(__uint_as_float(g[e]), __uint_as_float(g[e + 1]));
        x = __is_same(T, __half) ? __ffma2_rn(x, uu, dd) : __fadd2_rn(x, dd);
        x = __fmul2_rn(x, make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])));
        g[e] = __float_as_uint(x.x);
        g[e + 1] = __float_as_uint(x.y);
      }
      if (!whole) {                                    // unseen keys: whatever their S and dP are
#pragma unroll
        for (int e = 0; e < 64; ++e) g[e] = e < lim ? g[e] : 0u;
      }
      uint32_t ds[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) ds[e] = pack2(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]), T());
      tc_st32(at + 128, ds);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.ds_full));
    }
    if (n > 0) {
      mbar_wait(smem_u32(&sh.done), 0, dead);
      tc_fence_after();
    }
    const float f = *dead ? __int_as_float(0x7fffffff) : d.scale / up;
    T* out = attn_row<T>(d.dq, b, s.q0 + (row ? i : 0), row ? h : 0);
    float* part = a.q_splits > 1
                      ? a.part_q + (((int64_t)split * d.B * d.Hkv + head) * ((int64_t)d.Lq * G) + m) * d.D
                      : nullptr;
#pragma unroll
    for (int q = 0; q < DP / 2; q += 32) {
      const int c0 = w * (DP / 2) + q;
      if (c0 < d.D) write32<T>(quarter + 256 + c0, n > 0, f, out, part, d.D, c0, row, base + warp * 2048);   // (the rings are idle)
    }
  }
  finish(sh, d.status, warp, n > 0);
}

// ---------------------------------------------------------------- dk, dv
// Tensor memory: S^T, dP^T, dv, dk; P^T overwrites S^T and dS^T dP^T, each half in place.  While the groups are
// at P of tile t, the tensor cores are at dk of tile t - 1 and dP of tile t; while they are at dS of t, at
// dv of t and S of t + 1.  Up to a head size of 64 there is room for two of S^T, and S of t + 1 starts
// before P of t is there (the groups waited 750 of 2600 cycles for it).  Measured on one B200: 2 x 4096 causal, 32/8 heads
// of 128, 436 us (1260 TFLOP/s over the four products, tensor pipe 71 % busy: K and V are left operands in shared
// memory, since the accumulators fill tensor memory); 20 packed sequences of up to 1025, 16 heads of 64, 178 us.
template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 1) k_attn_dkv(const __grid_constant__ BwdArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  constexpr int kBlocks = DP / 64, kTile = kBlocks * kBlockBytes;
  constexpr bool kBf = __is_same(T, __nv_bfloat16);
  constexpr int kS = DP == 64 ? 2 : 1, kDp = kS * 128, kDv = kDp + 128, kDk = kDv + DP;   // S's buffers; columns
  const uint32_t sk = smem_u32(base), sv = sk + kTile;
  Shared& sh = *reinterpret_cast<Shared*>(base + (2 + a.q_stages + a.go_stages) * kTile);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
  const b3r_attention_desc& d = a.d;
  const int G = a.G, split = blockIdx.x % a.k_splits;
  int head, tile;
  place(blockIdx.x / a.k_splits, a.k_tiles, a.group, d.B * d.Hkv, false, head, tile);
  const int b = head / d.Hkv, kv = head % d.Hkv;
  const AttnSeq s = attn_seq(d, b);
  const int j0 = tile * kTileRows, keys = d.cu_k ? s.kl : d.Lk;
  if (j0 >= keys) return;
  // query tiles from the first that sees this tile's first key, of each head in turn
  int t0 = 0, per_head = 0, first = 0, n = 0;
  if (j0 < s.kl) {
    t0 = d.causal ? max(0, j0 - (s.kl - s.ql)) / kTileRows : 0;
    per_head = max(0, (s.ql + kTileRows - 1) / kTileRows - t0);
    const int all = per_head * G, per = (all + a.k_splits - 1) / a.k_splits;
    first = split * per;
    n = min(max(all - first, 0), per);
  }
  if (threadIdx.x == 0) init_shared(sh);
  if (warp == 9 && n > 0) tc_alloc(smem_u32(&sh.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  volatile int* dead = &sh.dead;
  const int steps = (d.D + 15) / 16;
  Ring qr{sk + 2 * kTile, base + 2 * kTile, sh.full[0], sh.empty[0], a.q_stages};
  Ring gr{sk + (2 + a.q_stages) * kTile, base + (2 + a.q_stages) * kTile, sh.full[1], sh.empty[1], a.go_stages};

  if (warp >= 8) {
    few_registers();
    if (warp == 8 && n > 0) {
    int fixes = 0;
    const int bk = d.cu_k ? 0 : b, bq = d.cu_q ? 0 : b;
    if (lane == 0) {
      const uint32_t bar = smem_u32(&sh.own_full);
      mbar_expect(bar, 2 * kTile);
#pragma unroll
      for (int c = 0; c < kBlocks; ++c) {
        tma_box(sk + c * kBlockBytes, &a.k, c * 64, (int)s.k0 + j0, kv, bk, bar);
        tma_box(sv + c * kBlockBytes, &a.v, c * 64, (int)s.k0 + j0, kv, bk, bar);
      }
    }
    int h = kv * G + first / per_head, t = first % per_head;
    for (int it = 0; it < n; ++it) {
      const int i0 = (t0 + t) * kTileRows;
      // P and dS are zero past the last query and meet the rows of dO and Q there
      if (a.lose && blockIdx.x + it == 0) qr.step();   // (a test: it never comes)
      else ring_load<kBlocks, kTileRows>(qr, &a.q, (int)s.q0 + i0, h, bq, s.ql - i0, true, &sh.fix, fixes, lane, dead);
      ring_load<kBlocks, kTileRows>(gr, &a.go, (int)s.q0 + i0, h, bq, s.ql - i0, true, &sh.fix, fixes, lane, dead);
      if (++t == per_head) {
        t = 0;
        ++h;
      }
    }
    if (*dead && lane == 0) mbar_wait(smem_u32(&sh.own_full), 0, dead);
  } else if (warp == 9 && n > 0) {
    {
      const uint32_t on = elect_one();
      const uint32_t id_s = mma_idesc(kBf, 128, 128, false), id_o = mma_idesc(kBf, 128, (d.D + 15) & ~15, true);
      auto product = [&](uint32_t acc, uint32_t left, uint32_t right) {   // acc = K Q^T or V dO^T
        tile_product<kBlocks, kTileRows>(acc, left, right, id_s, steps, on);
      };
      int xq, xg, last_round = 0;
      const uint64_t weights = desc_step(smem_u32(sh.weights)), minus = desc_step(smem_u32(sh.stat));
      auto scores = [&](int it) {
        xq = qr.next(dead);
        mbar_wait(smem_u32(&sh.st_full[it & (kPlain - 1)]), (it / kPlain) & 1, dead);
        product(tmem + it % kS * 128, sk, qr.data + xq * kTile);
        tc_mma(tmem + it % kS * 128, weights, minus + ((it & 1) * 2 * kStepBytes >> 4), id_s, true, on);
        tc_commit(smem_u32(&sh.s_full[it % kS]), on);
      };
      auto grads = [&](int it) {
        last_round = gr.round;
        xg = gr.next(dead);
        product(tmem + kDp, sv, gr.data + xg * kTile);
        tc_mma(tmem + kDp, weights, minus + (((it & 1) * 2 + 1) * kStepBytes >> 4), id_s, true, on);
        tc_commit(smem_u32(&sh.dp_full), on);
        tc_commit(smem_u32(&sh.st_empty[it & 1]), on);
      };
      mbar_wait(smem_u32(&sh.own_full), 0, dead);
      tc_fence_after();
      scores(0);
      grads(0);
      for (int it = 0; it < n; ++it) {
        const int cq = xq, cg = xg, round_g = last_round;
        if (kS == 2 && it + 1 < n) scores(it + 1);
        mbar_wait(smem_u32(&sh.p_full), it & 1, dead);
        tc_fence_after();
        tile_gather<kTileRows>(tmem + kDv, tmem + it % kS * 128, 64, gr.data + cg * kTile, id_o, it > 0, on);             // dv += P^T dO
        tc_commit(smem_u32(&sh.empty[1][cg]), on);
        if (kS == 1 && it + 1 < n) scores(it + 1);
        mbar_wait(smem_u32(&sh.ds_full), it & 1, dead);
        tc_fence_after();
        tile_gather<kTileRows>(tmem + kDk, tmem + kDp, 64, qr.data + cq * kTile, id_o, it > 0, on);  // dk += dS^T Q
        tc_commit(smem_u32(&sh.empty[0][cq]), on);
        if (it + 1 < n) {
          grads(it + 1);
        } else {
          tc_commit(smem_u32(&sh.done), on);
          mbar_wait(smem_u32(&sh.empty[1][cg]), round_g & 1, dead);     // no arrival is left behind
          mbar_wait(smem_u32(&sh.done), 0, dead);
        }
      }
    }
    } else if (warp == 10 && n > 0) {
    // the statistics of each tile's queries, two tiles ahead at most
    const bool apart = !kBf && a.far[head] != 0;
    {
      const uint32_t lo = pack2(weight_of(0), weight_of(1), T()), hi = pack2(weight_of(2), weight_of(3), T());
      for (int i = lane; i < kStepBytes / 16; i += 32) {               // bricks of 8: a step's first and second half by turns
        sh.weights[i] = (i & 8) ? make_uint4(0, 0, 0, 0) : make_uint4(lo, hi, 0, 0);
        for (int k = 0; k < 4; ++k)
          if (i & 8) sh.stat[k >> 1][k & 1][i] = make_uint4(0, 0, 0, 0);
      }
    }
    int h = kv * G + first / per_head, t = first % per_head;
    for (int it = 0; it < n; ++it) {
      const int st = it & 1, i0 = (t0 + t) * kTileRows;
      const float* l = attn_row<const float>(d.lse, b, s.q0 + i0, h);
      const float* dl = a.delta + ((int64_t)b * d.Hq + h) * d.Lq + i0;
      float x[4], y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool ok = i0 + q * 32 + lane < s.ql;
        x[q] = ok ? l[(q * 32 + lane) * d.lse.row] : -INFINITY;
        y[q] = ok ? dl[q * 32 + lane] : 0.f;
      }
      if (it >= 2) mbar_wait(smem_u32(&sh.st_empty[st]), ((it >> 1) - 1) & 1, dead);
      const int pl = it & (kPlain - 1);   // (free: st_empty of it - 2 follows dP of that tile, asked for after dS of it - 3)
      auto put = [&](int which, int row, float v) {
        float part[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          part[k] = f_of(t_of<T>(v * (1.f / weight_of(k))));
          v -= part[k] * weight_of(k);
        }
        sh.stat[st][which][(row >> 3) * 16 + (row & 7)] = make_uint4(pack2(part[0], part[1], T()), pack2(part[2], part[3], T()), 0, 0);
      };
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // a query that sees nothing, or none: its P is masked, or meets zeros; any low score will do
        const bool none = x[q] == -INFINITY;
        const float l_of = none ? -1e7f : shift_of<T>(x[q], d.scale), d_of = none ? 0.f : -y[q];
        if (apart) {
          sh.plain[pl][0][q * 32 + lane] = l_of;
          sh.plain[pl][1][q * 32 + lane] = d_of;
        }
        put(0, q * 32 + lane, apart ? 0.f : l_of);
        put(1, q * 32 + lane, apart ? 0.f : d_of);
      }
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.st_full[pl]));
      if (++t == per_head) {
        t = 0;
        ++h;
      }
    }
    }
  } else {
    many_registers();
    const int w = warp >> 2, r = threadIdx.x & 127, j = j0 + r;
    const bool row = j < keys;
    const uint32_t quarter = tmem + ((uint32_t)(warp & 3) << 21);
    const float c = d.scale * kLog2e;
    const float up = scale_ds<T>(a.range, head), down = up / kScaleP<T>;
    const float2 cc = make_float2(c, c), unscale = make_float2(down, down);
    const int see = d.causal ? max(0, j - (s.kl - s.ql)) : 0;         // the first query that sees this key
    // (two loops: the test within one cost float16 8 % of the kernel on sequences of a thousand)
    auto walk = [&](auto far) {
      int t = n > 0 ? first % per_head : 0;
      for (int it = 0; it < n; ++it) {
        const int i0 = (t0 + t) * kTileRows + w * 64;
        if (++t == per_head) t = 0;
        const uint32_t at = quarter + it % kS * 128 + w * 64, dp = quarter + kDp + w * 64;
        mbar_wait(smem_u32(&sh.s_full[it % kS]), (it / kS) & 1, dead);
        tc_fence_after();
        const int hide = see - i0;                                     // columns before it do not see the key
        const bool whole = __all_sync(0xffffffffu, hide <= 0);
        uint32_t p[64], g[64];
        auto add = [&](uint32_t (&to)[64], int which) {
          const float4* f = reinterpret_cast<const float4*>(&sh.plain[it & (kPlain - 1)][which][w * 64]);
#pragma unroll
          for (int e = 0; e < 64; e += 4) {
            const float4 z = f[e / 4];
            to[e] = __float_as_uint(__uint_as_float(to[e]) + z.x);
            to[e + 1] = __float_as_uint(__uint_as_float(to[e + 1]) + z.y);
            to[e + 2] = __float_as_uint(__uint_as_float(to[e + 2]) + z.z);
            to[e + 3] = __float_as_uint(__uint_as_float(to[e + 3]) + z.w);
          }
        };
        tc_ld32(at, p);
        tc_ld32(at + 32, p + 32);
        tc_wait_ld(p);
        if constexpr (decltype(far)::value) {
          mbar_wait(smem_u32(&sh.st_full[it & (kPlain - 1)]), (it / kPlain) & 1, dead);   // (there before S^T)
          add(p, 0);
        }
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 x = __fmul2_rn(make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])), cc);
          p[e] = __float_as_uint(ex2(x.x));
          p[e + 1] = __float_as_uint(ex2(x.y));
        }
        if (!whole) {                                                  // (apart: within the loops it doubled their time)
#pragma unroll
          for (int e = 0; e < 64; ++e) p[e] = e >= hide ? p[e] : 0u;
        }
        uint32_t h[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) h[e] = pack2(__uint_as_float(p[2 * e]), __uint_as_float(p[2 * e + 1]), T());
        tc_st32(at, h);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full));
        mbar_wait(smem_u32(&sh.dp_full), it & 1, dead);
        tc_fence_after();
        tc_ld32(dp, g);
        tc_ld32(dp + 32, g + 32);
        tc_wait_ld(g);
        if constexpr (decltype(far)::value) add(g, 1);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          float2 x = make_float2(__uint_as_float(g[e]), __uint_as_float(g[e + 1]));
          if (kScaleP<T> != 1.f) x = __fmul2_rn(x, unscale);
          x = __fmul2_rn(x, make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])));
          g[e] = __float_as_uint(x.x);
          g[e + 1] = __float_as_uint(x.y);
        }
        if (!whole) {                                                  // (dP may be anything there)
#pragma unroll
          for (int e = 0; e < 64; ++e) g[e] = e >= hide ? g[e] : 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) h[e] = pack2(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]), T());
        tc_st32(dp, h);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.ds_full));
      }
    };
    if (!kBf && a.far[head] != 0) walk(std::true_type());
    else walk(std::false_type());
    if (n > 0) {
      mbar_wait(smem_u32(&sh.done), 0, dead);
      tc_fence_after();
    }
    // one group writes dv, the other dk; keys past the sequence's end get zeros
    float f = w ? d.scale / up : 1.f / kScaleP<T>;
    if (*dead) f = __int_as_float(0x7fffffff);
    const bool has = n > 0;
    const b3r_attn_tensor& to = w ? d.dk : d.dv;
    T* out = attn_row<T>(to, b, s.k0 + (row ? j : 0), kv);
    float* part = a.k_splits > 1
                      ? a.part_k + ((((int64_t)split * 2 + w) * d.B * d.Hkv + head) * (int64_t)d.Lk + j) * d.D
                      : nullptr;
#pragma unroll
    for (int q = 0; q < DP; q += 32) {
      if (q >= d.D) break;
      // keys past the sequence's end get zeros, whatever their rows of the accumulators hold
      const uint32_t from = quarter + (w ? kDk : kDv) + q;
      uint8_t* const box = base + 2 * kTile + warp * 2048;             // (the rings are idle)
      if (__any_sync(0xffffffffu, row && j >= s.kl)) write32<T>(0, false, f, out, part, d.D, q, row && j >= s.kl, box);
      if (__any_sync(0xffffffffu, row && j < s.kl)) write32<T>(from, has, f, out, part, d.D, q, row && j < s.kl, box);
    }
  }
  finish(sh, d.status, warp, n > 0);
}

// Adds the float32 parts in their order.  One thread to four columns of a row; one pass over the parts.
// WHICH 0: dq (rows of queries x heads of a group); 1, 2: dv, dk.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_add(const __grid_constant__ BwdArgs a, int which) {
  const b3r_attention_desc& d = a.d;
  const int G = d.Hq / d.Hkv, head = blockIdx.y, b = head / d.Hkv, kv = head % d.Hkv, quads = d.D / 4;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, m = idx / quads;
  const int c = (int)(idx % quads) * 4;
  const AttnSeq s = attn_seq(d, b);
  const int64_t rows = which ? (int64_t)d.Lk : (int64_t)d.Lq * G;
  const int64_t mine = which ? (d.cu_k ? s.kl : d.Lk) : (int64_t)(d.cu_q ? s.ql : d.Lq) * G;
  if (m >= mine) return;
  const float* p = which ? a.part_k + (((int64_t)(which == 2) * d.B * d.Hkv + head) * rows + m) * d.D
                         : a.part_q + ((int64_t)head * rows + m) * d.D;
  const int64_t step = (which ? 2 : 1) * (int64_t)d.B * d.Hkv * rows * d.D;
  const int n = which ? a.k_splits : a.q_splits;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < n; ++i) {
    const float4 x = *reinterpret_cast<const float4*>(p + i * step + c);
    t.x += x.x;
    t.y += x.y;
    t.z += x.z;
    t.w += x.w;
  }
  T* out = which ? attn_row<T>(which == 2 ? d.dk : d.dv, b, s.k0 + m, kv)
                 : attn_row<T>(d.dq, b, s.q0 + m / G, kv * G + (int)(m % G));
  *reinterpret_cast<uint2*>(out + c) = make_uint2(pack2(t.x, t.y, T()), pack2(t.z, t.w, T()));
}

int64_t align256(int64_t b) { return (b + 255) & ~int64_t(255); }

int64_t cut(BwdArgs& a) {     // returns the workspace's bytes
  const b3r_attention_desc& d = a.d;
  const int64_t G = d.Hq / d.Hkv, heads = (int64_t)d.B * d.Hkv;
  a.q_tiles = (int)((d.Lq * G + kTileRows - 1) / kTileRows);
  a.k_tiles = (d.Lk + kTileRows - 1) / kTileRows;
  const int64_t q_blocks = a.q_tiles * heads, k_blocks = a.k_tiles * heads;
  const int64_t k_walk = (int64_t)((d.Lq + kTileRows - 1) / kTileRows) * G;   // query tiles that a key block meets
  // fewer blocks than SMs: the walk is split, at least two tiles to a block
  auto split = [](int64_t blocks, int64_t walk) {
    return blocks <= 0 || blocks >= kSms ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>((kSms + blocks - 1) / blocks, walk / 2));
  };
  a.q_splits = split(q_blocks, a.k_tiles);
  a.k_splits = split(k_blocks, k_walk);
  const int dp = d.D <= 64 ? 64 : 128, tile = dp / 64 * kBlockBytes;
  const int room = (232448 - 1024 - (int)sizeof(Shared)) / tile, stages = std::min(2 * kMaxStages, room - 2);
  a.q_stages = (stages + 1) / 2;   // Q is kept for longer than dO, and K than V
  a.go_stages = stages / 2;
  a.dq_k_stages = std::min(kMaxStages, (room + 1) / 2);
  a.dq_v_stages = std::min(kMaxStages, room / 2);
  a.q_tma = kTileRows % G == 0;
  a.G = (int)G;
  const int64_t head = std::max<int64_t>(1, ((int64_t)d.Lk + d.Lq * G) * d.D * 4);
  // Causal blocks differ by up to the whole length of a walk: the longest come first over all heads (in groups
  // of heads the last group's long ones ended late: 529 against 427 us for dk, dv at 4096 x 4096, 32/8 heads of 128).
  a.group = d.causal ? (int)std::max<int64_t>(1, heads) : (int)std::max<int64_t>(1, std::min<int64_t>(heads, (32 << 20) / head));
  int64_t n = align256((int64_t)d.B * d.Hq * d.Lq * 4);
  const int64_t r_off = n;
  if (d.dtype == B3R_F16) n += align256(heads * 12);
  const int64_t q_off = n;
  if (a.q_splits > 1) n += align256((int64_t)a.q_splits * heads * d.Lq * G * d.D * 4);
  const int64_t k_off = n;
  if (a.k_splits > 1) n += align256((int64_t)a.k_splits * 2 * heads * d.Lk * d.D * 4);
  uint8_t* w = reinterpret_cast<uint8_t*>(d.work);
  a.delta = reinterpret_cast<float*>(w);
  a.range = reinterpret_cast<float2*>(w + r_off);
  a.far = reinterpret_cast<int*>(a.range + heads);
  a.part_q = reinterpret_cast<float*>(w + q_off);
  a.part_k = reinterpret_cast<float*>(w + k_off);
  return n;
}

template <int DP, typename T>
int launch(const BwdArgs& a, cudaStream_t s) {
  const b3r_attention_desc& d = a.d;
  const int64_t G = d.Hq / d.Hkv, heads = (int64_t)d.B * d.Hkv;
  const int fixed = 1024 + (int)sizeof(Shared), tile = (DP / 64) * kBlockBytes;
  const int smem_q = fixed + (a.dq_k_stages + a.dq_v_stages) * tile, smem = fixed + (2 + a.q_stages + a.go_stages) * tile;
  B3R_REQUIRE(a.q_tiles * heads * a.q_splits <= 0x7fffffff && a.k_tiles * heads * a.k_splits <= 0x7fffffff,
              "attention backward: too many rows for one call");
  if constexpr (__is_same(T, __half)) {
    B3R_TRY(check_cuda(cudaMemsetAsync(a.range, 0, heads * 12, s), "attention backward"));
    const int64_t chunks = (std::max(d.Lq, d.Lk) + kRangeRows - 1) / kRangeRows;
    B3R_REQUIRE(chunks * d.B <= 0x7fffffff && d.Hq + d.Hkv <= 65535, "attention backward: too many rows for one call");
    if (chunks > 0) {
      k_attn_range<T><<<dim3((unsigned)(chunks * d.B), d.Hq + d.Hkv), 256, 0, s>>>(a, (int)chunks);
      B3R_TRY(check_launch("attention backward"));
    }
  }
  if (a.q_tiles > 0 && (!d.cu_q || d.Tq > 0)) {
    static uint64_t ready = 0;
    B3R_TRY(attn_smem(k_attn_dq<DP, T>, ready, "attention dq"));
    k_attn_dq<DP, T><<<(unsigned)(a.q_tiles * heads * a.q_splits), kThreads, smem_q, s>>>(a);
    B3R_TRY(check_launch("attention dq"));
    if (a.q_splits > 1) {
      k_attn_add<T><<<dim3((unsigned)((d.Lq * G * (d.D / 4) + 255) / 256), (unsigned)heads), 256, 0, s>>>(a, 0);
      B3R_TRY(check_launch("attention dq sum"));
    }
  }
  if (a.k_tiles > 0 && (!d.cu_k || d.Tk > 0)) {
    static uint64_t ready = 0;
    B3R_TRY(attn_smem(k_attn_dkv<DP, T>, ready, "attention dk, dv"));
    k_attn_dkv<DP, T><<<(unsigned)(a.k_tiles * heads * a.k_splits), kThreads, smem, s>>>(a);
    B3R_TRY(check_launch("attention dk, dv"));
    for (int which = 1; which <= 2 && a.k_splits > 1; ++which) {
      k_attn_add<T><<<dim3((unsigned)(((int64_t)d.Lk * (d.D / 4) + 255) / 256), (unsigned)heads), 256, 0, s>>>(a, which);
      B3R_TRY(check_launch("attention dk, dv sum"));
    }
  }
  return B3R_OK;
}

}  // namespace
}  // namespace b3r

using namespace b3r;

extern "C" int64_t b3r_attention_bwd_work_bytes(const b3r_attention_desc* d) {
  if (attn_check_sizes(d) != B3R_OK) return -1;
  if (d->B == 0) return 0;
  BwdArgs a;
  a.d = *d;
  return cut(a);
}

extern "C" int b3r_attention_bwd(const b3r_attention_desc* d, void* stream) { return b3r_attention_bwd_ex(d, 0, stream); }

extern "C" int b3r_attention_bwd_ex(const b3r_attention_desc* d, int flags, void* stream) {
  B3R_TRY(attn_check(d, true));
  B3R_REQUIRE((flags & ~B3R_ATTENTION_TEST_LOST_COPY) == 0, "attention backward: unknown flags");
  B3R_TRY(attn_clear(d, true, as_stream(stream)));
  if (d->B == 0) return B3R_OK;
  BwdArgs a;
  a.d = *d;
  a.lose = flags & B3R_ATTENTION_TEST_LOST_COPY;
  if (cut(a) > 0)
    B3R_REQUIRE(d->work && ((uintptr_t)d->work & 255) == 0, "attention backward: work buffer must be 256-byte aligned");
  const int64_t nq = d->cu_q ? d->Tq : d->Lq, nk = d->cu_q ? d->Tk : d->Lk;
  const int batch = d->cu_q ? 1 : d->B;
  B3R_TRY(attn_map(&a.q, d->q, nq, d->Hq, batch, d->D, d->dtype, kTileRows));
  B3R_TRY(attn_map(&a.go, d->d_o, nq, d->Hq, batch, d->D, d->dtype, kTileRows));
  B3R_TRY(attn_map(&a.k, d->k, nk, d->Hkv, batch, d->D, d->dtype, kTileRows));
  B3R_TRY(attn_map(&a.v, d->v, nk, d->Hkv, batch, d->D, d->dtype, kTileRows));
  if (a.q_tma) {
    B3R_TRY(attn_map_groups(&a.qg, d->q, nq, d->Hq, a.G, batch, d->D, d->dtype));
    B3R_TRY(attn_map_groups(&a.gog, d->d_o, nq, d->Hq, a.G, batch, d->D, d->dtype));
    B3R_TRY(attn_map_groups(&a.og, d->o, nq, d->Hq, a.G, batch, d->D, d->dtype));
  }
  cudaStream_t s = as_stream(stream);
  if (d->dtype == B3R_BF16) return d->D <= 64 ? launch<64, __nv_bfloat16>(a, s) : launch<128, __nv_bfloat16>(a, s);
  return d->D <= 64 ? launch<64, __half>(a, s) : launch<128, __half>(a, s);
}
