// Attention's forward pass on the 5th-generation tensor cores.
//
// Rows are (query, head of the group) pairs: row m of key/value head kv is query m / G with head
// kv G + m % G, so the heads that share keys and values fill one tile and read them once.  A
// block owns two tiles of 128 rows, or one where there are no more rows, and walks over tiles of
// keys:
//   warp 8    loads Q, K and V tiles by TMA, K and V into rings of stages
//   warp 9    issues S_w = Q_w K^T into one of the S buffers in tensor memory
//   warp 11   issues O_w += P_w V, P_w read from tensor memory (in one warp, issuing both took longer
//             than the products themselves: 2000 cycles a step against 750 to 1350)
//   warp 10   finds and decodes the block's next job
//   warps 0-3, 4-7: one group for each tile w; a thread owns a row, keeps its running maximum and
//             sum, and writes P_w as 16-bit pairs over S_w
// While one group is at its exponentials, the tensor cores work for the other.  With one tile of
// rows both groups share it and take every other key tile each; their parts are joined at the end.
// Few rows over many keys are split over blocks along the keys; a second kernel joins the parts.
//
// The maximum that the exponentials are taken against follows the true one only when it has
// grown by more than 2^8: P, its sum and O then carry the same factor, which cancels in O / l, so
// O in tensor memory is rescaled a few times at most instead of at every tile.  P is rounded to the
// operands' type for the product (its sum is taken before, in float32).  In float16 it is carried 2^7 times as large
// besides, 2^15 at most: keys that share little among many would else fall below float16's numbers (30000
// probabilities of 2^-25, which round to 2^-24, doubled what they add to o).
//
// What bounds it, measured on one B200 (1669 TFLOP/s, 6.5 TB/s):
//   one query over 32768 keys (16 sequences, 32/8 heads of 128): 228 us, 5.6 TB/s: HBM
//   769 x 769 (64 sequences, 16 heads of 64, float16): 406 us, 382 TFLOP/s: no pipe (exponentials busy 38 %, tensor cores
//     24 %).  A step of two tiles takes 2100 to 2500 cycles (its exponentials 2048, 16 a cycle and SM), a job's end
//     4000; tiles that 769 = 6 x 128 + 1 leaves nearly empty run alone; a third of a mean job's 29 thousand
//     cycles is not accounted for
//   16384 x 16384, causal, 16/4 heads of 128: 890 us in a burst, 1235 TFLOP/s (1030 to 1080 in a long run, at the power
//     limit): the products, 88 cycles for each 16 of the head size with Q in shared memory
// The softmax groups' 208 registers leave no room for what all roles share: 112 to 148 bytes of it lie in local memory,
// written once (without their code nothing spills; each other role accounts for some of the loads).
#include <algorithm>
#include "b3r_attn.cuh"
#include "b3r_tc.cuh"

namespace b3r {
namespace {

constexpr int kThreads = 384;   // three warpgroups: two of softmax, one of loads and products
constexpr int kMaxStages = 8;
constexpr int kAskAhead = 4;    // key tiles before its end at which a job's successor is asked for
constexpr float kGrow = 8.f;    // log2 of how far the maximum may grow before O is rescaled
template <typename T>
constexpr float kUp = __is_same(T, __half) ? 7.f : 0.f;   // log2 of P at the maximum that it is taken against

struct alignas(64) FwdArgs {
  CUtensorMap q, k, v;
  b3r_attention_desc d;
  int tiles;        // pairs of row tiles (single ones when `one`) of the longest sequence
  int one;          // one tile of rows: the groups share it and split the keys
  int splits;       // jobs along the keys
  int G, heads;     // query heads to a group; B x Hkv
  uint32_t g_mul, g_shift;   // for divisions by G
  int k_stages, v_stages, group;
  int q_tma;        // the heads of a group divide 128: Q comes by TMA, a box of whole groups
  int lose;         // a test: block 0 never gets its first keys
  float* part_o;    // [splits][B Hkv][rows][D]
  float* part_l;    // [splits][B Hkv][rows]: log2 of the sum, -inf where a part sees nothing
};

// Buffers of a head size.  Up to 64, tensor memory holds three buffers of S beside O, so that a
// group's next scores are ready when it ends the last ones, and shared memory two of Q.  Above, S has one
// for each group, and the next scores follow the product that reads P out of it; one warp issues
// both, so that no barrier lies between them (3430 cycles a step of both groups against 3800).  Two
// buffers of 64 keys instead took 4160: with its left operand in shared memory a product of N = 64
// takes as long as one of N = 128, about 100 cycles for each 16 of the head size.
template <int DP>
struct Cfg {
  static constexpr int kBlocks = DP / 64, kTile = kBlocks * kBlockBytes;
  static constexpr bool kOneIssuer = DP > 64;
  static constexpr int kS = kOneIssuer ? 2 : 3, kQ = kOneIssuer ? 1 : 2;
  static constexpr int kOut = kS * kTileRows;                              // O's first column
};
constexpr int kMaxS = 3;
constexpr int kStage = 32 * 64;   // bytes of a softmax warp's rows on their way out: 32 rows of 32 columns

// One job: two tiles of rows (one) of a key/value head, and a range of its keys.
struct Job {
  int b, kv, split;
  int q0, k0, ql, kl, rows;
  int m0[2];         // first row of each group's tile
  int first, n[2];   // first key tile, and how many each group takes; n[0] < 0: there are no more jobs
  int buf;           // S buffer of its first step
};

constexpr int kJobs = 3;   // jobs that a block has in hand at most

// The barriers of S and P are each group's own, one for each of its last kS steps: a group that takes
// no part in a job must not meet a barrier that has turned twice since.  Nor may it turn one for the other
// group, which it can be two jobs ahead of: where the groups write their rows of Q, each fills its own tile,
// on barriers and in an order of buffers of its own (q_full[w]), in the jobs that it takes part in alone.
struct Shared {
  uint64_t q_full[2][2], q_empty[2], fix, k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
  uint64_t s_full[2][kMaxS], p_full[2][kMaxS], s_free[kMaxS], o_done[2];
  uint64_t job_full[kJobs], job_empty[kJobs], want, cancel, half_full, half_free;
  alignas(16) uint4 answer;
  Job job[kJobs];
  uint32_t tmem;
  int dead;
  float m[kTileRows], l[kTileRows];   // of the second group, where both share a tile
};

__device__ __forceinline__ int div_g(const FwdArgs& a, int m) { return (int)((__umulhi((uint32_t)m, a.g_mul) + (uint32_t)m) >> a.g_shift); }

__device__ __forceinline__ void decode(const FwdArgs& a, int id, Job& j) {
  const b3r_attention_desc& d = a.d;
  j.split = id % a.splits;
  id /= a.splits;
  // heads in groups whose keys and values fit L2; within a group the row tiles with most work first
  const int gsz = a.group * a.tiles, g = id / gsz, r = id - g * gsz;
  const int width = min(a.group, a.heads - g * a.group);
  const int tile = a.tiles - 1 - r / width, head = g * a.group + r % width;
  j.b = head / d.Hkv;
  j.kv = head - j.b * d.Hkv;
  const AttnSeq s = attn_seq(d, j.b);
  j.q0 = (int)s.q0;
  j.k0 = (int)s.k0;
  j.ql = s.ql;
  j.kl = s.kl;
  j.rows = (d.cu_q ? s.ql : d.Lq) * a.G;
  const int seen = s.ql * a.G;
  int n[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    j.m0[w] = a.one ? tile * kTileRows : (2 * tile + w) * kTileRows;
    const int last = min(j.m0[w] + kTileRows, seen) - 1;
    n[w] = last < j.m0[w] ? 0 : (attn_bound(s, div_g(a, last), d.causal) + kTileRows - 1) / kTileRows;
  }
  const int all = max(n[0], n[1]), per = (all + a.splits - 1) / a.splits;
  j.first = j.split * per;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int mine = min(max(n[w] - j.first, 0), per);
    j.n[w] = a.one ? (mine + 1 - w) / 2 : mine;
  }
}

// Where row m of a job's tile goes.
template <typename T>
struct RowOut {
  T* o;
  float* lse;
  float *part_o, *part_l;
  __device__ __forceinline__ RowOut(const FwdArgs& a, const Job& j, int m) {
    const b3r_attention_desc& d = a.d;
    const int i = div_g(a, m), h = j.kv * a.G + m - i * a.G;
    o = attn_row<T>(d.o, j.b, (int64_t)j.q0 + i, h);
    lse = attn_row<float>(d.lse, j.b, (int64_t)j.q0 + i, h);
    const int64_t at = ((int64_t)j.split * a.heads + (int64_t)j.b * d.Hkv + j.kv) * ((int64_t)d.Lq * a.G) + m;
    part_o = a.part_o + at * d.D;
    part_l = a.part_l + at;
  }
};

// The next job of a block.  The grid has a block for every job; a block that runs takes jobs over from
// blocks that have not begun, so the barriers, tensor memory and loads of one serve many, and work of
// unequal lengths spreads by itself.  (One warp; returns -1 when there are none left.)
__device__ __forceinline__ void ask_next(Shared& sh) {
  mbar_expect(smem_u32(&sh.cancel), 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(&sh.answer)),
               "r"(smem_u32(&sh.cancel))
               : "memory");
}
__device__ __forceinline__ int read_next(Shared& sh) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, r;\n\t}"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(&sh.answer))
      : "memory");
  return ok ? (int)x : -1;
}

// A role's place in the block's list of jobs.
struct JobList {
  Shared& sh;
  int slot = 0, round = 0;
  __device__ __forceinline__ explicit JobList(Shared& s) : sh(s) {}
  // The next job, once it is there; nullptr after the last.
  __device__ __forceinline__ const Job* get(volatile int* dead) {
    mbar_wait(smem_u32(&sh.job_full[slot]), round & 1, dead);
    return __any_sync(0xffffffffu, sh.job[slot].n[0] < 0 || *dead) ? nullptr : &sh.job[slot];
  }
  // Ends the role's use of it (one lane of a warp that has read all it needs).
  __device__ __forceinline__ void done(int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.job_empty[slot]));
    if (++slot == kJobs) {
      slot = 0;
      ++round;
    }
  }
};

// Issuing warp: waits for a job's tiles of Q, and where they are.  By TMA both come to the job's buffer; else each
// group that takes part has filled the next one of its own.
template <int DP>
struct QTiles {
  uint32_t at[2];
  int turns[2] = {0, 0};   // jobs of the block (by TMA), or that a group has taken part in
  __device__ __forceinline__ void get(const FwdArgs& a, Shared& sh, uint32_t sq, int n0, int n1, volatile int* dead) {
    using X = Cfg<DP>;
    const uint32_t q_bytes = (a.one ? 1 : 2) * X::kTile;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (w == 1 && (a.one || a.q_tma)) {
        at[1] = a.one ? at[0] : at[0] + X::kTile;
      } else if (a.q_tma || (w ? n1 : n0) > 0) {
        const int buf = turns[w] % X::kQ;
        mbar_wait(smem_u32(&sh.q_full[w][buf]), (turns[w] / X::kQ) & 1, dead);
        at[w] = sq + buf * q_bytes + w * X::kTile;
        ++turns[w];
      }
    }
  }
};

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 1) k_attn_fwd(const __grid_constant__ FwdArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  using X = Cfg<DP>;
  constexpr int kTile = X::kTile;
  constexpr bool kBf = __is_same(T, __nv_bfloat16);
  const int q_tiles = a.one ? 1 : 2, q_bytes = q_tiles * kTile;
  const uint32_t sq = smem_u32(base), sk = sq + X::kQ * q_bytes, sv = sk + a.k_stages * kTile;
  uint8_t* const stage = base + X::kQ * q_bytes + (a.k_stages + a.v_stages) * kTile;
  Shared& sh = *reinterpret_cast<Shared*>(stage + 8 * kStage);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
  const b3r_attention_desc& d = a.d;
  if (warp == 9) tc_alloc(smem_u32(&sh.tmem), 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      for (int w = 0; w < 2; ++w) mbar_init(smem_u32(&sh.q_full[w][i]), a.q_tma ? 1 : 4);   // (by TMA: q_full[0], both tiles)
      mbar_init(smem_u32(&sh.q_empty[i]), 1);
      mbar_init(smem_u32(&sh.o_done[i]), 1);
    }
    mbar_init(smem_u32(&sh.fix), 1);
    for (int i = 0; i < a.k_stages; ++i) {
      mbar_init(smem_u32(&sh.k_full[i]), 1);
      mbar_init(smem_u32(&sh.k_empty[i]), 1);
      mbar_init(smem_u32(&sh.v_full[i]), 1);
      mbar_init(smem_u32(&sh.v_empty[i]), 1);
    }
    for (int i = 0; i < kMaxS; ++i) {
      for (int w = 0; w < 2; ++w) {
        mbar_init(smem_u32(&sh.s_full[w][i]), 1);
        mbar_init(smem_u32(&sh.p_full[w][i]), 4);
      }
      mbar_init(smem_u32(&sh.s_free[i]), 1);
    }
    for (int i = 0; i < kJobs; ++i) {
      mbar_init(smem_u32(&sh.job_full[i]), 1);
      mbar_init(smem_u32(&sh.job_empty[i]), X::kOneIssuer ? 10 : 11);   // loads, products, eight softmax warps
    }
    mbar_init(smem_u32(&sh.want), 1);
    mbar_init(smem_u32(&sh.cancel), 1);
    mbar_init(smem_u32(&sh.half_full), 4);
    mbar_init(smem_u32(&sh.half_free), 4);
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
    if (warp == 8) {
      // ------------------------------------------------ loads
      Ring kr{sk, base + X::kQ * q_bytes, sh.k_full, sh.k_empty, a.k_stages};
      Ring vr{sv, base + X::kQ * q_bytes + a.k_stages * kTile, sh.v_full, sh.v_empty, a.v_stages};
      int fixes = 0, k = 0;
      JobList list(sh);
      while (const Job* j = list.get(dead)) {
        if (a.q_tma) {                         // rows past the end only reach their own scores
          const int qb = k % X::kQ, use = k / X::kQ;
          const uint32_t bar = smem_u32(&sh.q_full[0][qb]);
          const bool free = use == 0 || mbar_wait(smem_u32(&sh.q_empty[qb]), (use - 1) & 1, dead);
          if (free && lane == 0) {
            mbar_expect(bar, q_bytes);
            for (int w = 0; w < q_tiles; ++w)
#pragma unroll
              for (int c = 0; c < X::kBlocks; ++c)
                tma_box(sq + qb * q_bytes + w * kTile + c * kBlockBytes, &a.q, c * 64, j->kv * a.G, j->q0 + div_g(a, j->m0[w]),
                        d.cu_q ? 0 : j->b, bar);
          }
        }
        const int tiles = a.one ? j->n[0] + j->n[1] : max(j->n[0], j->n[1]);
        const int ask = max(0, tiles - kAskAhead), batch = d.cu_k ? 0 : j->b;
        for (int i = 0; i < tiles; ++i) {
          const int row = (j->first + i) * kTileRows;
          if (i == ask && lane == 0) mbar_arrive(smem_u32(&sh.want));   // near the job's end: the next one, not sooner
          if (a.lose && blockIdx.x == 0 && k + i == 0) kr.step();   // (a test: these keys never come)
          else ring_load<X::kBlocks, kTileRows>(kr, &a.k, j->k0 + row, j->kv, batch, j->kl - row, false, &sh.fix, fixes, lane, dead);
          // P is zero past the last key, so V is cleared there
          ring_load<X::kBlocks, kTileRows>(vr, &a.v, j->k0 + row, j->kv, batch, j->kl - row, true, &sh.fix, fixes, lane, dead);
        }
        list.done(lane);
        ++k;
      }
    } else if (X::kOneIssuer && warp == 9) {
      // ------------------------------------------------ scores and outputs, S_w = Q_w K^T after O_w += P_w V
      const uint32_t on = elect_one();
      const uint32_t id_s = mma_idesc(kBf, 128, kTileRows, false), id_o = mma_idesc(kBf, 128, (d.D + 15) & ~15, true);
      const int steps = (d.D + 15) / 16;
      const uint32_t bar_s = smem_u32(sh.s_full), bar_p = smem_u32(sh.p_full), bar_o = smem_u32(sh.o_done);
      const uint32_t bar_k = smem_u32(sh.k_empty), bar_v = smem_u32(sh.v_empty);
      Ring kr{sk, base + X::kQ * q_bytes, sh.k_full, sh.k_empty, a.k_stages};
      Ring vr{sv, base + X::kQ * q_bytes + a.k_stages * kTile, sh.v_full, sh.v_empty, a.v_stages};
      int hs0 = 0, hs1 = 0, ts0 = 0, ts1 = 0;   // each group's steps whose S, and O, has been issued
      QTiles<DP> q;
      int last = -1, last_round = 0;
      JobList list(sh);
      while (const Job* j = list.get(dead)) {
        const int n0 = j->n[0], n1 = j->n[1], n = max(n0, n1);
        list.done(lane);
        q.get(a, sh, sq, n0, n1, dead);
        auto scores = [&](int w, int& hs, int st) {
          tc_fence_after();
          tile_product<X::kBlocks, kTileRows>(tmem + w * kTileRows, q.at[w], sk + st * kTile, id_s, steps, on);
          tc_commit(bar_s + (w * kMaxS + (hs & 1)) * 8, on);
          ++hs;
        };
        auto output = [&](int w, int& ts, int st, bool add) {
          mbar_wait(bar_p + (w * kMaxS + (ts & 1)) * 8, (ts >> 1) & 1, dead);
          tc_fence_after();
          tile_gather<kTileRows>(tmem + X::kOut + w * DP, tmem + w * kTileRows, 32, sv + st * kTile, id_o, add, on);
          tc_commit(bar_o + w * 8, on);
          ++ts;
        };
        auto next_v = [&]() {
          last_round = vr.round;
          return last = vr.next(dead);
        };
        int st = 0, sw = 0;
        if (!a.one) st = kr.next(dead);
        if (n0 > 0) {
          if (a.one) st = kr.next(dead);
          scores(0, hs0, st);
          if (a.one) tc_commit(bar_k + st * 8, on);
        }
        if (n1 > 0) {
          if (a.one) st = kr.next(dead);
          scores(1, hs1, st);
          if (a.one) tc_commit(bar_k + st * 8, on);
        }
        if (!a.one) tc_commit(bar_k + st * 8, on);
        for (int i = 0; i < n; ++i) {
          if (!a.one) {
            sw = next_v();
            if (i + 1 < n) st = kr.next(dead);
          }
          auto group = [&](int w, int nw, int& hs, int& ts) {
            if (i >= nw) return;
            if (a.one) sw = next_v();
            output(w, ts, sw, i > 0);
            if (a.one) tc_commit(bar_v + sw * 8, on);
            if (i + 1 >= nw) return;
            if (a.one) st = kr.next(dead);
            scores(w, hs, st);
            if (a.one) tc_commit(bar_k + st * 8, on);
          };
          group(0, n0, hs0, ts0);
          group(1, n1, hs1, ts1);
          if (!a.one) {
            if (i + 1 < n) tc_commit(bar_k + st * 8, on);
            tc_commit(bar_v + sw * 8, on);
          }
          if (i + 2 == n || n == 1) tc_commit(smem_u32(&sh.q_empty[0]), on);   // the last scores are on their way
        }
      }
      if (last >= 0) mbar_wait(bar_v + last * 8, last_round & 1, dead);   // no arrival is left behind
    } else if (!X::kOneIssuer && warp == 9) {
      // ------------------------------------------------ scores: S = Q_w K^T, step by step
      const uint32_t on = elect_one(), id_s = mma_idesc(kBf, 128, kTileRows, false);
      const int steps = (d.D + 15) / 16;
      const uint32_t bar_s = smem_u32(sh.s_full), bar_f = smem_u32(sh.s_free), bar_e = smem_u32(sh.k_empty);
      Ring kr{sk, base + X::kQ * q_bytes, sh.k_full, sh.k_empty, a.k_stages};
      int k = 0, buf = 0, uses = 0, b0 = 0, b1 = 0;    // S buffer and its turn; each group's barrier
      int last_buf = -1, last_use = 0;
      QTiles<DP> q_at;
      JobList list(sh);
      while (const Job* j = list.get(dead)) {
        const int n0 = j->n[0], n1 = j->n[1], n = max(n0, n1), qb = k % X::kQ;
        list.done(lane);
        q_at.get(a, sh, sq, n0, n1, dead);
        const uint32_t q0 = q_at.at[0], q1 = q_at.at[1];
        auto product = [&](uint32_t q, int w, int& b, int st) {
          if (uses > 0) mbar_wait(bar_f + buf * 8, (uses - 1) & 1, dead);   // until P has been read from it
          tc_fence_after();
          tile_product<X::kBlocks, kTileRows>(tmem + buf * kTileRows, q, sk + st * kTile, id_s, steps, on);
          tc_commit(bar_s + (w * kMaxS + b) * 8, on);
          b = b + 1 == X::kS ? 0 : b + 1;
          last_buf = buf;
          last_use = uses;
          if (++buf == X::kS) {
            buf = 0;
            ++uses;
          }
        };
        for (int i = 0; i < n; ++i) {
          int st = 0;
          if (!a.one) st = kr.next(dead);
          if (i < n0) {
            if (a.one) st = kr.next(dead);
            product(q0, 0, b0, st);
            if (a.one) tc_commit(bar_e + st * 8, on);
          }
          if (i < n1) {
            if (a.one) st = kr.next(dead);
            product(q1, 1, b1, st);
            if (a.one) tc_commit(bar_e + st * 8, on);
          }
          if (!a.one) tc_commit(bar_e + st * 8, on);
        }
        tc_commit(smem_u32(&sh.q_empty[qb]), on);
        ++k;
      }
      // no arrival is left behind: the last step's P is read after all that was issued here
      if (last_buf >= 0) mbar_wait(bar_f + last_buf * 8, last_use & 1, dead);
    } else if (!X::kOneIssuer && warp == 11) {
      // ------------------------------------------------ outputs: O_w += P V, step by step
      const uint32_t on = elect_one(), id_o = mma_idesc(kBf, 128, (d.D + 15) & ~15, true);
      const uint32_t bar_p = smem_u32(sh.p_full), bar_f = smem_u32(sh.s_free), bar_o = smem_u32(sh.o_done), bar_e = smem_u32(sh.v_empty);
      Ring vr{sv, base + X::kQ * q_bytes + a.k_stages * kTile, sh.v_full, sh.v_empty, a.v_stages};
      int buf = 0, b0 = 0, b1 = 0, r0 = 0, r1 = 0;     // P's buffer; each group's barrier and its round
      int last = -1, last_round = 0;
      JobList list(sh);
      while (const Job* j = list.get(dead)) {
        const int n0 = j->n[0], n1 = j->n[1], n = max(n0, n1);
        list.done(lane);
        auto product = [&](int w, int& b, int& r, int st, bool add) {
          mbar_wait(bar_p + (w * kMaxS + b) * 8, r & 1, dead);
          tc_fence_after();
          tile_gather<kTileRows>(tmem + X::kOut + w * DP, tmem + buf * kTileRows, 32, sv + st * kTile, id_o, add, on);
          tc_commit(bar_o + w * 8, on);
          tc_commit(bar_f + buf * 8, on);
          if (++b == X::kS) {
            b = 0;
            ++r;
          }
          buf = buf + 1 == X::kS ? 0 : buf + 1;
        };
        for (int i = 0; i < n; ++i) {
          int st = 0;
          auto next = [&]() {
            last_round = vr.round;
            last = st = vr.next(dead);
          };
          if (!a.one) next();
          if (i < n0) {
            if (a.one) next();
            product(0, b0, r0, st, i > 0);
            if (a.one) tc_commit(bar_e + st * 8, on);
          }
          if (i < n1) {
            if (a.one) next();
            product(1, b1, r1, st, i > 0);
            if (a.one) tc_commit(bar_e + st * 8, on);
          }
          if (!a.one) tc_commit(bar_e + st * 8, on);
        }
      }
      if (last >= 0) mbar_wait(bar_e + last * 8, last_round & 1, dead);   // no arrival is left behind
    } else if (warp == 10) {
      // ------------------------------------------------ jobs
      int id = blockIdx.x, slot = 0, round = 0, buf = 0, asks = 0;
      for (int k = 0;;) {
        Job j;
        if (id >= 0) {
          decode(a, id, j);
          if (j.m0[0] < j.rows && j.n[0] + j.n[1] == 0) {   // rows that see nothing: cleared here and now
            const int last = min(j.m0[a.one ? 0 : 1] + kTileRows, j.rows);
            for (int m = j.m0[0]; m < last; ++m) {
              const RowOut<T> to(a, j, m);
              if (a.splits > 1) {
                if (lane == 0) *to.part_l = -INFINITY;   // the part itself is not read then
              } else {
                for (int c = lane * 8; c < d.D; c += 256) *reinterpret_cast<uint4*>(to.o + c) = make_uint4(0, 0, 0, 0);
                if (lane == 0) *to.lse = -INFINITY;
              }
            }
          }
        } else {
          j.n[0] = j.n[1] = -1;
        }
        if (id < 0 || j.n[0] + j.n[1] > 0) {
          const bool free = round == 0 || mbar_wait(smem_u32(&sh.job_empty[slot]), (round - 1) & 1, dead);
          if (__any_sync(0xffffffffu, !free || *dead)) break;   // (the others see it for themselves)
          j.buf = buf;
          if (lane == 0) {
            sh.job[slot] = j;
            mbar_arrive(smem_u32(&sh.job_full[slot]));
          }
          __syncwarp();
          if (id < 0) break;
          buf = (buf + j.n[0] + j.n[1]) % X::kS;
          if (++slot == kJobs) {
            slot = 0;
            ++round;
          }
          mbar_wait(smem_u32(&sh.want), k & 1, dead);    // until the loads are near its end
          ++k;
        }
        if (lane == 0) ask_next(sh);
        __syncwarp();
        const bool told = mbar_wait(smem_u32(&sh.cancel), asks & 1, dead);
        ++asks;
        id = __all_sync(0xffffffffu, told) ? read_next(sh) : -1;
        fence_async();                                   // the answer is read before the next one is written
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------ softmax, one row to a thread
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t quarter = tmem + ((uint32_t)(warp & 3) << 21);   // this warp's 32 lanes
    const float c = d.scale * kLog2e;
    int mine = 0, turn = 0;                    // this group's steps so far; the jobs that it has written Q for
    JobList list(sh);
    for (int k = 0;; ++k) {
      const Job* jp = list.get(dead);
      if (!jp) break;
      const Job& j = *jp;
      const int n = j.n[w], n0 = j.n[0], n1 = j.n[1], buf0 = j.buf, first = j.first;
      const int m = j.m0[a.one ? 0 : w] + r;
      const bool row = m < j.rows;
      const int i = div_g(a, m);
      AttnSeq sq_;
      sq_.ql = j.ql;
      sq_.kl = j.kl;
      // (past the rows nothing is written: such a thread sees what lets its warp take whole tiles)
      const int bound = !row ? j.kl : i < j.ql ? attn_bound(sq_, i, d.causal) : 0;
      if (!a.q_tma && n > 0 && (w == 0 || !a.one)) {
        // the row of Q into the swizzled tile; zeros past D and past the rows
        const int h = j.kv * a.G + m - i * a.G;
        const uint4* q = reinterpret_cast<const uint4*>(attn_row<const T>(d.q, j.b, (int64_t)j.q0 + (row ? i : 0), row ? h : 0));
        uint8_t* dst = base + (turn % X::kQ) * q_bytes + w * kTile + r * 128;
#pragma unroll
        for (int cb = 0; cb < DP / 8; ++cb) {
          const uint4 x = (row && cb * 8 < d.D) ? q[cb] : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(dst + (cb >> 3) * kBlockBytes + (((cb & 7) ^ (r & 7)) << 4)) = x;
        }
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[w][turn % X::kQ]));
        ++turn;
      }
      const bool any = __any_sync(0xffffffffu, row);   // a warp without rows only keeps the others' pace
      float mx = -INFINITY, l = 0.f;       // what the exponentials are taken against (log2), and their sum
      for (int it = 0; it < n; ++it, ++mine) {
        // the step's place among all steps of the block gives its buffer
        const int g = buf0 + min(it, n0) + min(it, n1) + (w && it < n0), bar = mine % X::kS;
        const uint32_t at = quarter + (X::kOneIssuer ? w : g % X::kS) * kTileRows;
        const int lim = bound - (first + (a.one ? 2 * it + w : it)) * kTileRows;   // keys of this tile that the row sees
        mbar_wait(smem_u32(&sh.s_full[w][bar]), (mine / X::kS) & 1, dead);
        tc_fence_after();
        if (!any) {
          if (mine > 0) mbar_wait(smem_u32(&sh.o_done[w]), (mine - 1) & 1, dead);   // (every turn is met)
          if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[w][bar]));
          continue;
        }
        auto follow = [&](float top) {                   // moves mx after the true maximum (2^kUp below it), O and l with it
          const bool grow = top > mx + (kGrow + kUp<T>) || mx == -INFINITY;   // (mx = -inf: nothing summed yet)
          if (it > 0 && __any_sync(0xffffffffu, grow && top > mx)) {
            const float f = grow && top > mx ? ex2(mx - (top - kUp<T>)) : 1.f;      // 0 for the first key that the row sees
            mbar_wait(smem_u32(&sh.o_done[w]), (mine - 1) & 1, dead);
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < DP; q += 32) {
              uint32_t o[32];
              tc_ld32(quarter + X::kOut + w * DP + q, o);
              tc_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tc_st32(quarter + X::kOut + w * DP + q, o);
            }
            l *= f;
          }
          if (grow) mx = top - kUp<T>;
        };
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto exps = [&](const uint32_t* s, uint32_t to) {   // 32 columns of P
          const float2 cc = make_float2(c, c), mm = make_float2(mx == -INFINITY ? 0.f : -mx, mx == -INFINITY ? 0.f : -mx);
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), cc, mm);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum[e & 1] = __fadd2_rn(sum[e & 1], x);
            p[e] = pack2(x.x, x.y, T());
          }
          tc_st16(to, p);
        };
        if (__all_sync(0xffffffffu, lim >= kTileRows)) {
          uint32_t s[kTileRows];
#pragma unroll
          for (int q = 0; q < kTileRows; q += 32) tc_ld32(at + q, s + q);
          tc_wait_ld(s);
          float t[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] = fmaxf(__uint_as_float(s[e]), __uint_as_float(s[4 + e]));
#pragma unroll
          for (int q = 8; q < kTileRows; q += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = fmaxf(fmaxf(t[e], __uint_as_float(s[q + e])), __uint_as_float(s[q + 4 + e]));
          follow(fmaxf(mx, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * c));
#pragma unroll
          for (int q = 0; q < kTileRows; q += 32) exps(s + q, at + q / 2);
        } else {
          // a tile that ends inside: 32 columns at a time, up to the last one that a row of the warp sees (in a body of
          // its own, 421 us for 64 x 769 x 769 and 16 heads of 64; with masks in one body for all tiles 441, and
          // with branches around each half of one body 445)
          const int end = __reduce_max_sync(0xffffffffu, lim);
          float t = -INFINITY;
          uint32_t s[32];
          auto some = [&](int q) {
            tc_ld32(at + q, s);
            tc_wait_ld(s);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e] = q + e < lim ? s[e] : 0xff800000u;
          };
#pragma unroll 1
          for (int q = 0; q < min(end, kTileRows); q += 32) {
            some(q);
#pragma unroll
            for (int e = 0; e < 32; ++e) t = fmaxf(t, __uint_as_float(s[e]));
          }
          follow(fmaxf(mx, t * c));
#pragma unroll 1
          for (int q = 0; q < kTileRows; q += 32) {
            if (q < end) {
              some(q);                                   // (P only overwrites scores that have been read)
              exps(s, at + q / 2);
            } else {
              uint32_t p[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) p[e] = 0;
              tc_st16(at + q / 2, p);
            }
          }
        }
        tc_wait_st();
        // the last step's product ends long before, but has to be seen: o_done's turns are met one by one
        if (mine > 0) mbar_wait(smem_u32(&sh.o_done[w]), (mine - 1) & 1, dead);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[w][bar]));
        sum[0] = __fadd2_rn(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      const RowOut<T> to(a, j, row ? m : 0);
      if (n > 0) {
        mbar_wait(smem_u32(&sh.o_done[w]), (mine - 1) & 1, dead);
        tc_fence_after();
      }
      // ---------------------------------------------- output
      float f0 = 0.f, f1 = 0.f, lg;                      // factors of O (and of the other group's O); log2 of the sum
      if (a.one) {
        if (w == 1) {
          sh.m[r] = mx;
          sh.l[r] = l;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.half_full));
        } else {
          mbar_wait(smem_u32(&sh.half_full), k & 1, dead);
          tc_fence_after();
          const float m1 = sh.m[r], l1 = sh.l[r], top = fmaxf(mx, m1);
          const float e0 = mx == -INFINITY ? 0.f : ex2(mx - top), e1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
          const float sum = l * e0 + l1 * e1;
          f0 = sum > 0.f ? e0 / sum : 0.f;
          f1 = sum > 0.f ? e1 / sum : 0.f;
          lg = sum != 0.f ? top + __log2f(sum) : -INFINITY;
          if (isnan(sum)) f0 = f1 = lg = sum;
        }
      } else {
        f0 = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;     // NaN stays NaN
        lg = l == 0.f ? -INFINITY : mx + __log2f(l);
      }
      if (w == 0 || !a.one) {
        const bool has0 = n > 0 && any, has1 = a.one && n1 > 0 && any;
        if (*dead) f0 = f1 = lg = __int_as_float(0x7fffffff);
#pragma unroll
        for (int q = 0; q < DP; q += 32) {
          if (q >= d.D) break;
          uint32_t o[32];
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
          if (has0) {
            tc_ld32(quarter + X::kOut + w * DP + q, o);
            tc_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]) * f0;
          }
          if (has1) {
            tc_ld32(quarter + X::kOut + DP + q, o);
            tc_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += __uint_as_float(o[e]) * f1;
          }
          if (lg == -INFINITY)                           // a row that sees nothing
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.f;
          if (a.splits > 1) {
            if (row)
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                if (q + e < d.D) *reinterpret_cast<float4*>(to.part_o + q + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          } else {
            // through shared memory, so that four lanes write the 64 bytes of a row (a lane to a row took
            // 2500 to 4000 cycles a job); chunk c of row x lies at c ^ (x / 2 % 4), out of banks' way
            uint4* const box = reinterpret_cast<uint4*>(stage + warp * kStage);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              box[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_uint4(pack2(v[8 * e], v[8 * e + 1], T()), pack2(v[8 * e + 2], v[8 * e + 3], T()),
                                                                   pack2(v[8 * e + 4], v[8 * e + 5], T()), pack2(v[8 * e + 6], v[8 * e + 7], T()));
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              const int y = x + (lane >> 2), c = lane & 3;
              T* const out = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, row ? reinterpret_cast<uint64_t>(to.o) : 0, y));
              const uint4 z = box[y * 4 + (c ^ ((y >> 1) & 3))];
              if (out && q + c * 8 < d.D) *reinterpret_cast<uint4*>(out + q + c * 8) = z;
            }
          }
        }
        if (row) {
          if (a.splits > 1) *to.part_l = lg;
          else *to.lse = lg * kLn2;
        }
      }
      tc_fence_before();
      if (a.one) {                                       // the second group's O and sums have been read
        __syncwarp();
        if (w == 0 && lane == 0) mbar_arrive(smem_u32(&sh.half_free));
        if (w == 1) mbar_wait(smem_u32(&sh.half_free), k & 1, dead);
        tc_fence_after();
      }
      list.done(lane);
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

// Joins the parts of a row: weights 2^(lg_s - max) over their sum.  A part that is NaN (its scores were, or a wait
// ran out) makes the row NaN; the maximum would pass over it.  One warp to a row.  Latency bounds it: 5 us for
// 96 rows of 64 in 6 parts, 6 us for 512 rows of 128 in 5.
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
  bool nan = false;
  for (int p = lane; p < a.splits; p += 32) {
    const float lg = a.part_l[p * step + at];
    top = fmaxf(top, lg);
    nan = nan || isnan(lg);
  }
  nan = __any_sync(0xffffffffu, nan);
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
  if (nan) sum = __int_as_float(0x7fffffff);
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  const int i = (int)(m / G), h = kv * G + (int)(m % G);
  if (c < d.D)
    *reinterpret_cast<uint2*>(attn_row<T>(d.o, b, s.q0 + i, h) + c) =
        make_uint2(pack2(o.x * inv, o.y * inv, T()), pack2(o.z * inv, o.w * inv, T()));
  if (lane == 0) *attn_row<float>(d.lse, b, s.q0 + i, h) = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
}

// How the work is cut, from the descriptor alone (the lengths on the device are not known here).
void cut(FwdArgs& a) {
  const b3r_attention_desc& d = a.d;
  a.G = d.Hq / d.Hkv;
  a.heads = d.B * d.Hkv;
  // m / G = (umulhi(m, mul) + m) >> shift for 0 <= m < 2^31 (Granlund and Montgomery's division by an invariant)
  a.g_shift = 0;
  while ((1u << a.g_shift) < (uint32_t)a.G) ++a.g_shift;
  a.g_mul = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << a.g_shift) - a.G)) / a.G + 1);
  const int64_t rows = (int64_t)d.Lq * a.G;
  a.one = rows <= kTileRows;
  const int64_t job_rows = a.one ? kTileRows : 2 * kTileRows;
  a.tiles = (int)((rows + job_rows - 1) / job_rows);
  const int64_t jobs = (int64_t)a.tiles * d.B * d.Hkv, keys = (d.Lk + kTileRows - 1) / kTileRows;
  // Fewer jobs than SMs leave SMs idle: the keys are split, two tiles to a job at least (one for
  // each group).  Sequences of different lengths make some of these jobs shorter, so long key
  // ranges (8 tiles a job at least) are split into about four jobs an SM.
  a.splits = 1;
  if (jobs < kSms) a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(kSms / jobs, keys / 2));
  if (jobs < 4 * kSms && a.one)
    a.splits = (int)std::max<int64_t>(a.splits, std::min<int64_t>((4 * kSms + jobs - 1) / jobs, keys / 8));
  const int fixed = 1024 + 8 * kStage + (int)sizeof(Shared), q_tiles = a.one ? 1 : 2;
  const int room = d.D <= 64 ? (232448 - fixed) / Cfg<64>::kTile - Cfg<64>::kQ * q_tiles
                             : (232448 - fixed) / Cfg<128>::kTile - Cfg<128>::kQ * q_tiles;
  const int stages = std::min(2 * kMaxStages, room);
  a.k_stages = (stages + 1) / 2;       // K is needed first
  a.v_stages = stages / 2;
  // heads whose keys and values are at work at the same time: about 32 MB of the 126 MB L2
  const int64_t head = std::max<int64_t>(1, (int64_t)d.Lk * d.D * 4);
  a.group = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)d.B * d.Hkv, (32 << 20) / head));
}

template <int DP, typename T>
int launch(FwdArgs& a, cudaStream_t s) {
  const int smem = 1024 + Cfg<DP>::kQ * (a.one ? 1 : 2) * Cfg<DP>::kTile + (a.k_stages + a.v_stages) * Cfg<DP>::kTile + 8 * kStage +
                   (int)sizeof(Shared);
  static uint64_t ready = 0;
  B3R_TRY(attn_smem(k_attn_fwd<DP, T>, ready, "attention"));
  const int64_t jobs = (int64_t)a.tiles * a.heads * a.splits;
  B3R_REQUIRE(jobs <= 0x3fffffff, "attention: too many rows for one call");
  k_attn_fwd<DP, T><<<(unsigned)jobs, kThreads, smem, s>>>(a);
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

extern "C" int b3r_attention_fwd(const b3r_attention_desc* d, void* stream) { return b3r_attention_fwd_ex(d, 0, stream); }

extern "C" int b3r_attention_fwd_ex(const b3r_attention_desc* d, int flags, void* stream) {
  B3R_TRY(attn_check(d, false));
  B3R_REQUIRE((flags & ~B3R_ATTENTION_TEST_LOST_COPY) == 0, "attention: unknown flags");
  B3R_TRY(attn_clear(d, false, as_stream(stream)));
  if (d->B == 0 || d->Lq == 0 || (d->cu_q && d->Tq == 0)) return B3R_OK;
  FwdArgs a;
  a.d = *d;
  cut(a);
  a.lose = flags & B3R_ATTENTION_TEST_LOST_COPY;
  if (a.splits > 1) {
    B3R_REQUIRE(d->work && ((uintptr_t)d->work & 255) == 0, "attention: work buffer must be 256-byte aligned");
    a.part_o = reinterpret_cast<float*>(d->work);
    a.part_l = a.part_o + part_rows(a) * d->D;
  }
  B3R_TRY(attn_map(&a.k, d->k, d->cu_q ? d->Tk : d->Lk, d->Hkv, d->cu_q ? 1 : d->B, d->D, d->dtype, kTileRows));
  B3R_TRY(attn_map(&a.v, d->v, d->cu_q ? d->Tk : d->Lk, d->Hkv, d->cu_q ? 1 : d->B, d->D, d->dtype, kTileRows));
  const int G = d->Hq / d->Hkv;
  a.q_tma = kTileRows % G == 0;
  if (a.q_tma)
    B3R_TRY(attn_map_groups(&a.q, d->q, d->cu_q ? d->Tq : d->Lq, d->Hq, G, d->cu_q ? 1 : d->B, d->D, d->dtype));
  cudaStream_t s = as_stream(stream);
  if (d->dtype == B3R_BF16) return d->D <= 64 ? launch<64, __nv_bfloat16>(a, s) : launch<128, __nv_bfloat16>(a, s);
  return d->D <= 64 ? launch<64, __half>(a, s) : launch<128, __half>(a, s);
}
