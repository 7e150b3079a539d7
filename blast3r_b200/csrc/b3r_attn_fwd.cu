// Attention's forward pass on the 5th-generation tensor cores.
//
// Rows are (query, head of the group) pairs: row m of key/value head kv is query m / G with head
// kv G + m % G, so the heads that share keys and values fill one tile and read them once.  A
// block owns two tiles of 128 rows, or one where there are no more rows, and walks over tiles of
// 128 keys:
//   warp 8    loads K and V tiles by TMA into a ring of stages
//   warp 9    issues S_w = Q_w K^T (tensor memory) and O_w += P_w V, P_w read from tensor memory
//   warps 0-3, 4-7: one group for each tile w; a thread owns a row, keeps its running maximum and
//             sum, and writes P_w as 16-bit pairs over S_w
// While one group is at its exponentials, the tensor cores work for the other.  With one tile of
// rows both groups share it and take every other key tile each; their parts are joined at the end.
// Few rows over many keys are split over blocks along the keys; a second kernel joins the parts.
//
// The maximum that the exponentials are taken against follows the true one only when it has
// grown by more than 2^8: P, its sum and O then carry the same factor, which cancels in O / l, so
// O in tensor memory is rescaled a few times at most instead of at every tile.  P is rounded to the
// operands' type for the product (its sum is taken before, in float32).
#include <algorithm>
#include "b3r_attn.cuh"
#include "b3r_tc.cuh"

namespace b3r {
namespace {

constexpr int kThreads = 384;   // three warpgroups: two of softmax, one of loads and products
constexpr int kMaxStages = 8;
constexpr float kGrow = 8.f;   // log2 of how far the maximum may grow before O is rescaled

struct alignas(64) FwdArgs {
  CUtensorMap q, k, v;
  b3r_attention_desc d;
  int tiles;        // pairs of row tiles (single ones when `one`) of the longest sequence
  int one;          // one tile of rows: the groups share it and split the keys
  int splits;       // blocks along the keys
  int stages, group;
  int q_tma;        // the heads of a group divide 128: Q comes by TMA, a box of whole groups
  float* part_o;    // [splits][B Hkv][rows][D]
  float* part_l;    // [splits][B Hkv][rows]: log2 of the sum, -inf where a part sees nothing
};

struct Shared {
  uint64_t q_full, fix, kv_full[kMaxStages], kv_empty[kMaxStages], s_full[2], p_full[2], o_done[2];
  uint32_t tmem;
  int dead;
  float m[kTileRows], l[kTileRows];
};

// What a block works on; the same in every role.
struct Job {
  AttnSeq s;
  int b, kv, split, rows, G;
  int m0[2];     // first row of each group's tile
  int first, n[2];   // first key tile, and how many each group takes
};

__device__ __forceinline__ Job job_of(const FwdArgs& a) {
  const b3r_attention_desc& d = a.d;
  Job j;
  const int heads = d.B * d.Hkv;
  int id = blockIdx.x;
  j.split = id % a.splits;
  id /= a.splits;
  // heads in groups whose keys and values fit L2; within a group the row tiles with most work first
  const int gsz = a.group * a.tiles, g = id / gsz, r = id - g * gsz;
  const int width = min(a.group, heads - g * a.group);
  const int tile = a.tiles - 1 - r / width, head = g * a.group + r % width;
  j.b = head / d.Hkv;
  j.kv = head % d.Hkv;
  j.G = d.Hq / d.Hkv;
  j.s = attn_seq(d, j.b);
  j.rows = (d.cu_q ? j.s.ql : d.Lq) * j.G;
  const int seen = j.s.ql * j.G;
  int n[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    j.m0[w] = a.one ? tile * kTileRows : (2 * tile + w) * kTileRows;
    const int last = min(j.m0[w] + kTileRows, seen) - 1;
    n[w] = last < j.m0[w] ? 0 : (attn_bound(j.s, last / j.G, d.causal) + kTileRows - 1) / kTileRows;
  }
  const int all = max(n[0], n[1]), per = (all + a.splits - 1) / a.splits;
  j.first = j.split * per;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int mine = min(max(n[w] - j.first, 0), per);
    j.n[w] = a.one ? (mine + 1 - w) / 2 : mine;
  }
  return j;
}

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 1) k_attn_fwd(const __grid_constant__ FwdArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  constexpr int kBlocks = DP / 64, kTile = kBlocks * kBlockBytes;
  constexpr bool kBf = sizeof(T) == 2 && __is_same(T, __nv_bfloat16);
  const int q_tiles = a.one ? 1 : 2;
  const uint32_t sq = smem_u32(base), skv = sq + q_tiles * kTile;
  Shared& sh = *reinterpret_cast<Shared*>(base + (q_tiles + a.stages) * kTile);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
  if (warp == 9) tc_alloc(smem_u32(&sh.tmem), 512);   // first: it takes longer than the rest of the set-up
  const Job j = job_of(a);
  const b3r_attention_desc& d = a.d;
  const bool idle = j.m0[0] >= j.rows;                // no rows of this sequence here
  const bool none = idle || j.n[0] + j.n[1] == 0;
  const uint32_t bar_q = smem_u32(&sh.q_full);
  if (threadIdx.x == 0) {
    mbar_init(bar_q, a.q_tma ? 1 : 8);
    mbar_init(smem_u32(&sh.fix), 1);
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(smem_u32(&sh.kv_full[i]), 1);
      mbar_init(smem_u32(&sh.kv_empty[i]), 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&sh.s_full[w]), 1);
      mbar_init(smem_u32(&sh.p_full[w]), 4);
      mbar_init(smem_u32(&sh.o_done[w]), 1);
    }
    sh.dead = 0;
    fence_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  volatile int* dead = &sh.dead;
  // a softmax thread holds a row of 128 scores: registers move over from the third warpgroup
  // (256 x 208 + 128 x 88 = 384 x 168, what the block was launched with)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8 && !none) {
    // ------------------------------------------------ loads
    Ring ring{skv, base + q_tiles * kTile, sh.kv_full, sh.kv_empty, a.stages};
    int fixes = 0;
    if (a.q_tma && lane == 0) {        // whole groups of heads fill a tile: rows past the end only reach their own scores
      mbar_expect(bar_q, q_tiles * kTile);
      for (int w = 0; w < q_tiles; ++w)
#pragma unroll
        for (int c = 0; c < kBlocks; ++c)
          tma_box(sq + w * kTile + c * kBlockBytes, &a.q, c * 64, j.kv * j.G, (int)j.s.q0 + j.m0[w] / j.G, d.cu_q ? 0 : j.b, bar_q);
    }
    const int row0 = (int)j.s.k0, batch = d.cu_k ? 0 : j.b;
    auto load = [&](const CUtensorMap* map, int tile, bool values) {   // P is zero past the last key, so V is cleared there
      ring_load<kBlocks>(ring, map, row0 + tile * kTileRows, j.kv, batch, j.s.kl - tile * kTileRows, values, &sh.fix, fixes, lane,
                         dead);
    };
    if (a.one) {
      for (int w = 0; w < 2; ++w)
        if (j.n[w] > 0) load(&a.k, j.first + w, false);
      for (int i = 0; i < j.n[0]; ++i)
        for (int w = 0; w < 2; ++w) {
          if (i < j.n[w]) load(&a.v, j.first + 2 * i + w, true);
          if (i + 1 < j.n[w]) load(&a.k, j.first + 2 * (i + 1) + w, false);
        }
    } else {
      const int n = max(j.n[0], j.n[1]);
      load(&a.k, j.first, false);
      for (int i = 0; i < n; ++i) {
        load(&a.v, j.first + i, true);
        if (i + 1 < n) load(&a.k, j.first + i + 1, false);
      }
    }
    } else if (warp == 9 && !none) {
    // ------------------------------------------------ matrix products
    {
      const uint32_t on = elect_one();
      const uint32_t id_s = mma_idesc(kBf, 128, 128, false), id_o = mma_idesc(kBf, 128, (d.D + 15) & ~15, true);
      const int steps = (d.D + 15) / 16;
      Ring ring{skv, base + q_tiles * kTile, sh.kv_full, sh.kv_empty, a.stages};
      int last = 0, last_round = 0;
      auto next = [&]() {
        last_round = ring.round;
        return last = ring.next(dead);
      };
      auto scores = [&](int w, int s) {                // S_w = Q_w K^T
        const uint32_t q = sq + (a.one ? 0 : w) * kTile, k = skv + s * kTile;
        tile_product<kBlocks>(tmem + w * 128, q, k, id_s, steps, on);
        tc_commit(smem_u32(&sh.s_full[w]), on);
      };
      auto output = [&](int w, int s, int i) {         // O_w += P_w V
        mbar_wait(smem_u32(&sh.p_full[w]), i & 1, dead);
        tc_fence_after();
        tile_gather(tmem + 256 + w * DP, tmem + w * 128, 32, skv + s * kTile, id_o, i > 0, on);
        tc_commit(smem_u32(&sh.o_done[w]), on);
      };
      auto release = [&](int s) { tc_commit(smem_u32(&sh.kv_empty[s]), on); };
      mbar_wait(bar_q, 0, dead);
      tc_fence_after();
      if (a.one) {
        for (int w = 0; w < 2; ++w)
          if (j.n[w] > 0) {
            const int s = next();
            scores(w, s);
            release(s);
          }
        for (int i = 0; i < j.n[0]; ++i)
          for (int w = 0; w < 2; ++w) {
            if (i < j.n[w]) {
              const int s = next();
              output(w, s, i);
              release(s);
            }
            if (i + 1 < j.n[w]) {
              const int s = next();
              scores(w, s);
              release(s);
            }
          }
      } else {
        const int n = max(j.n[0], j.n[1]);
        int sk = next();
        for (int w = 0; w < 2; ++w)
          if (j.n[w] > 0) scores(w, sk);
        release(sk);
        for (int i = 0; i < n; ++i) {
          const int sv = next();
          sk = i + 1 < n ? next() : -1;
          for (int w = 0; w < 2; ++w) {
            if (i < j.n[w]) output(w, sv, i);
            if (i + 1 < j.n[w]) scores(w, sk);
          }
          release(sv);
          if (sk >= 0) release(sk);
        }
      }
      mbar_wait(smem_u32(&sh.kv_empty[last]), last_round & 1, dead);   // no arrival is left behind
    }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------ softmax, one row to a thread
    const int w = warp >> 2, r = threadIdx.x & 127;
    const int m = j.m0[a.one ? 0 : w] + r;
    const int i = m / j.G, h = j.kv * j.G + m % j.G;
    const bool row = m < j.rows;
    const int bound = row && i < j.s.ql ? attn_bound(j.s, i, d.causal) : 0;
    const uint32_t quarter = tmem + ((uint32_t)(warp & 3) << 21);   // this warp's 32 lanes
    const float c = d.scale * kLog2e;
    if (!none && !a.q_tma) {
      if (w == 0 || !a.one) {
        // the row of Q into the swizzled tile; zeros past D and past the rows
        const uint4* q = reinterpret_cast<const uint4*>(attn_row<const T>(d.q, j.b, j.s.q0 + (row ? i : 0), row ? h : 0));
        uint8_t* dst = base + w * kTile + r * 128;
#pragma unroll
        for (int cb = 0; cb < DP / 8; ++cb) {
          const uint4 x = (row && cb * 8 < d.D) ? q[cb] : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(dst + (cb >> 3) * kBlockBytes + (((cb & 7) ^ (r & 7)) << 4)) = x;
        }
        fence_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q);
    }
    float mx = -INFINITY, l = 0.f;       // what the exponentials are taken against (log2), and their sum
    const int n = j.n[w];
    for (int it = 0; it < n; ++it) {
      const int lim = bound - (j.first + (a.one ? 2 * it + w : it)) * kTileRows;   // keys of this tile that the row sees
      mbar_wait(smem_u32(&sh.s_full[w]), it & 1, dead);
      tc_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int q = 0; q < 4; ++q) tc_ld32(quarter + w * 128 + q * 32, s + q * 32);
      tc_wait_ld(s);
      if (!__all_sync(0xffffffffu, lim >= kTileRows)) {
#pragma unroll
        for (int q = 0; q < 128; ++q) s[q] = q < lim ? s[q] : 0xff800000u;
      }
      float t0 = __uint_as_float(s[0]), t1 = __uint_as_float(s[1]);
#pragma unroll
      for (int q = 2; q < 128; q += 2) {
        t0 = fmaxf(t0, __uint_as_float(s[q]));
        t1 = fmaxf(t1, __uint_as_float(s[q + 1]));
      }
      const float top = fmaxf(mx, fmaxf(t0, t1) * c);
      const bool grow = top > mx + kGrow || mx == -INFINITY;   // (mx = -inf: nothing summed yet)
      if (it > 0 && __any_sync(0xffffffffu, grow && top > mx)) {
        const float f = grow && top > mx ? ex2(mx - top) : 1.f;      // 0 for the first key that the row sees
        mbar_wait(smem_u32(&sh.o_done[w]), (it - 1) & 1, dead);
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < DP; q += 32) {
          uint32_t o[32];
          tc_ld32(quarter + 256 + w * DP + q, o);
          tc_wait_ld(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tc_st32(quarter + 256 + w * DP + q, o);
        }
        l *= f;
      }
      if (grow) mx = top;
      const float2 cc = make_float2(c, c), mm = make_float2(mx == -INFINITY ? 0.f : -mx, mx == -INFINITY ? 0.f : -mx);
      float2 sum = make_float2(0.f, 0.f);
      uint32_t p[64];
#pragma unroll
      for (int q = 0; q < 64; ++q) {
        float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), cc, mm);
        x.x = ex2(x.x);
        x.y = ex2(x.y);
        sum = __fadd2_rn(sum, x);
        p[q] = pack2(x.x, x.y, T());
      }
      tc_st32(quarter + w * 128, p);
      tc_st32(quarter + w * 128 + 32, p + 32);
      l += sum.x + sum.y;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[w]));
    }
    if (n > 0) {
      mbar_wait(smem_u32(&sh.o_done[w]), (n - 1) & 1, dead);
      tc_fence_after();
    }
    // ---------------------------------------------- output
    float f0 = 0.f, f1 = 0.f, lg;                      // factors of O (and of the other group's O); log2 of the sum
    if (a.one) {
      if (w == 1) {
        sh.m[r] = mx;
        sh.l[r] = l;
      }
      bar_sync(1, 256);
      if (w == 0) {
        const float m1 = sh.m[r], l1 = sh.l[r], top = fmaxf(mx, m1);
        const float e0 = mx == -INFINITY ? 0.f : ex2(mx - top), e1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
        const float sum = l * e0 + l1 * e1;
        f0 = sum > 0.f ? e0 / sum : 0.f;
        f1 = sum > 0.f ? e1 / sum : 0.f;
        lg = top + __log2f(sum);
        if (!(sum != 0.f)) lg = -INFINITY;
        if (isnan(sum)) f0 = f1 = lg = sum;
      }
      tc_fence_after();
    } else {
      f0 = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;     // NaN stays NaN
      lg = l == 0.f ? -INFINITY : mx + __log2f(l);
    }
    if (!idle && (w == 0 || !a.one)) {
      const bool has0 = n > 0, has1 = a.one && j.n[1] > 0;
      const int64_t at = ((int64_t)j.split * d.B * d.Hkv + (int64_t)j.b * d.Hkv + j.kv) * ((int64_t)d.Lq * j.G) + m;
      if (*dead) f0 = f1 = lg = __int_as_float(0x7fffffff);
#pragma unroll
      for (int q = 0; q < DP; q += 32) {
        if (q >= d.D) break;
        uint32_t o[32];
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.f;
        if (has0) {
          tc_ld32(quarter + 256 + w * DP + q, o);
          tc_wait_ld(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]) * f0;
        }
        if (has1) {
          tc_ld32(quarter + 256 + DP + q, o);
          tc_wait_ld(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] += __uint_as_float(o[e]) * f1;
        }
        if (lg == -INFINITY)                           // a row that sees nothing
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        if (!row) continue;
        if (a.splits > 1) {
          float* out = a.part_o + at * d.D + q;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (q + e < d.D) *reinterpret_cast<float4*>(out + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        } else {
          T* out = attn_row<T>(d.o, j.b, j.s.q0 + i, h) + q;
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (q + e < d.D)
              *reinterpret_cast<uint4*>(out + e) = make_uint4(pack2(v[e], v[e + 1], T()), pack2(v[e + 2], v[e + 3], T()),
                                                              pack2(v[e + 4], v[e + 5], T()), pack2(v[e + 6], v[e + 7], T()));
        }
      }
      if (row) {
        if (a.splits > 1) a.part_l[at] = lg;
        else *attn_row<float>(d.lse, j.b, j.s.q0 + i, h) = lg * kLn2;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*dead) {                                         // copies that a failed wait left behind
    for (int t = 0; t < 100; ++t) __nanosleep(1000);
    if (threadIdx.x == 0 && d.status) *d.status = 1;
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after();
    tc_free(tmem, 512);
  }
}

// Joins the parts of a row: weights 2^(lg_s - max) over their sum.  One warp to a row.
template <typename T>
__global__ void __launch_bounds__(128) k_attn_join(const __grid_constant__ FwdArgs a) {
  const b3r_attention_desc& d = a.d;
  const int G = d.Hq / d.Hkv, lane = threadIdx.x & 31;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int head = blockIdx.y, b = head / d.Hkv, kv = head % d.Hkv;
  const AttnSeq s = attn_seq(d, b);
  if (m >= (int64_t)(d.cu_q ? s.ql : d.Lq) * G) return;
  const int64_t rows = (int64_t)d.Lq * G, step = (int64_t)d.B * d.Hkv * rows, at = head * rows + m;
  float top = -INFINITY;
  for (int p = lane; p < a.splits; p += 32) top = fmaxf(top, a.part_l[p * step + at]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const int c = lane * 4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  if (top != -INFINITY)
    for (int p = 0; p < a.splits; ++p) {
      const float lg = a.part_l[p * step + at];
      if (lg == -INFINITY) continue;
      const float f = ex2(lg - top);
      sum += f;
      if (c < d.D) {
        const float4 x = *reinterpret_cast<const float4*>(a.part_o + (p * step + at) * d.D + c);
        o.x += f * x.x;
        o.y += f * x.y;
        o.z += f * x.z;
        o.w += f * x.w;
      }
    }
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  const int i = (int)(m / G), h = kv * G + (int)(m % G);
  if (c < d.D)
    *reinterpret_cast<uint2*>(attn_row<T>(d.o, b, s.q0 + i, h) + c) =
        make_uint2(pack2(o.x * inv, o.y * inv, T()), pack2(o.z * inv, o.w * inv, T()));
  if (lane == 0) *attn_row<float>(d.lse, b, s.q0 + i, h) = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
}

constexpr int kSms = 148;

// How the work is cut, from the descriptor alone (the lengths on the device are not known here).
void cut(FwdArgs& a) {
  const b3r_attention_desc& d = a.d;
  const int64_t rows = (int64_t)d.Lq * (d.Hq / d.Hkv);
  a.one = rows <= kTileRows;
  a.tiles = a.one ? 1 : (int)((rows + 2 * kTileRows - 1) / (2 * kTileRows));
  const int64_t blocks = (int64_t)a.tiles * d.B * d.Hkv, keys = (d.Lk + kTileRows - 1) / kTileRows;
  // Fewer blocks than SMs leave SMs idle: the keys are split, two tiles to a block at least (one
  // for each group).  Sequences of different lengths make some of these blocks shorter, so long
  // key ranges (8 tiles a block at least) are split into about four blocks an SM.
  a.splits = 1;
  if (blocks < kSms) a.splits = (int)std::max<int64_t>(1, std::min<int64_t>((kSms + blocks - 1) / blocks, keys / 2));
  if (blocks < 4 * kSms && a.one)
    a.splits = (int)std::max<int64_t>(a.splits, std::min<int64_t>((4 * kSms + blocks - 1) / blocks, keys / 8));
  const int dp = d.D <= 64 ? 64 : 128, tile = dp / 64 * kBlockBytes;
  a.stages = std::min(kMaxStages, (232448 - 1024 - (int)sizeof(Shared)) / tile - (a.one ? 1 : 2));
  // heads whose keys and values are at work at the same time: about 32 MB of the 126 MB L2
  const int64_t head = std::max<int64_t>(1, (int64_t)d.Lk * d.D * 4);
  a.group = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)d.B * d.Hkv, (32 << 20) / head));
}

template <int DP, typename T>
int launch(const FwdArgs& a, cudaStream_t s) {
  const int tile = DP / 64 * kBlockBytes;
  const int smem = 1024 + ((a.one ? 1 : 2) + a.stages) * tile + (int)sizeof(Shared);
  B3R_TRY(check_cuda(cudaFuncSetAttribute(k_attn_fwd<DP, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "attention"));
  const int64_t blocks = (int64_t)a.tiles * a.d.B * a.d.Hkv * a.splits;
  B3R_REQUIRE(blocks <= 0x7fffffff, "attention: too many rows for one call");
  k_attn_fwd<DP, T><<<(unsigned)blocks, kThreads, smem, s>>>(a);
  B3R_TRY(check_launch("attention"));
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.d.Lq * (a.d.Hq / a.d.Hkv);
    k_attn_join<T><<<dim3((unsigned)((rows + 3) / 4), a.d.B * a.d.Hkv), 128, 0, s>>>(a);
    B3R_TRY(check_launch("attention join"));
  }
  return B3R_OK;
}

}  // namespace
}  // namespace b3r

using namespace b3r;

static int64_t part_rows(const FwdArgs& a) { return (int64_t)a.splits * a.d.B * a.d.Lq * a.d.Hq; }

extern "C" int64_t b3r_attention_fwd_work_bytes(const b3r_attention_desc* d) {
  if (attn_check_sizes(d) != B3R_OK) return -1;
  if (d->B == 0 || d->Lq == 0) return 0;
  FwdArgs a;
  a.d = *d;
  cut(a);
  return a.splits > 1 ? part_rows(a) * (d->D + 1) * 4 : 0;
}

extern "C" int b3r_attention_fwd(const b3r_attention_desc* d, void* stream) {
  B3R_TRY(attn_check(d, false));
  if (d->B == 0 || d->Lq == 0 || (d->cu_q && d->Tq == 0)) return B3R_OK;
  FwdArgs a;
  a.d = *d;
  cut(a);
  if (a.splits > 1) {
    B3R_REQUIRE(d->work && ((uintptr_t)d->work & 255) == 0, "attention: work buffer must be 256-byte aligned");
    a.part_o = reinterpret_cast<float*>(d->work);
    a.part_l = a.part_o + part_rows(a) * d->D;
  }
  B3R_TRY(attn_map(&a.k, d->k, d->cu_q ? d->Tk : d->Lk, d->Hkv, d->cu_q ? 1 : d->B, d->D, d->dtype));
  B3R_TRY(attn_map(&a.v, d->v, d->cu_q ? d->Tk : d->Lk, d->Hkv, d->cu_q ? 1 : d->B, d->D, d->dtype));
  const int G = d->Hq / d->Hkv;
  a.q_tma = kTileRows % G == 0;
  if (a.q_tma)
    B3R_TRY(attn_map_groups(&a.q, d->q, d->cu_q ? d->Tq : d->Lq, d->Hq, G, d->cu_q ? 1 : d->B, d->D, d->dtype));
  cudaStream_t s = as_stream(stream);
  if (d->dtype == B3R_BF16) return d->D <= 64 ? launch<64, __nv_bfloat16>(a, s) : launch<128, __nv_bfloat16>(a, s);
  return d->D <= 64 ? launch<64, __half>(a, s) : launch<128, __half>(a, s);
}
