// Part 5 of the C ABI: attention's argument checks and its backward pass, with P = exp(S - lse):
//   delta = do . o,  dv = P^T do,  dP = do v^T,  dS = P (dP - delta),  dq = scale dS k,  dk = scale dS^T q
// A warp owns a row: a query row forward and for dq, a key row for dk and dv, which walks over the
// queries of all heads that share it.  Lanes own keys (queries) for the scores and
// dimensions for the sums, all in float32.
#include <algorithm>
#include "b3r_attn.cuh"

namespace b3r {

int attn_check_sizes(const b3r_attention_desc* d) {
  B3R_REQUIRE(d, "attention: NULL descriptor");
  B3R_REQUIRE(d->dtype == B3R_BF16 || d->dtype == B3R_F16, "attention: dtype must be bf16 or f16");
  B3R_REQUIRE(d->B >= 0 && d->Lq >= 0 && d->Lk >= 0 && d->Tq >= 0 && d->Tk >= 0, "attention: negative size");
  B3R_REQUIRE(d->D >= 8 && d->D <= 128 && d->D % 8 == 0, "attention: the head size is a multiple of 8 up to 128, got %d", d->D);
  B3R_REQUIRE(d->Hq >= 1 && d->Hkv >= 1 && d->Hq % d->Hkv == 0, "attention: %d query heads do not share %d key/value heads evenly",
              d->Hq, d->Hkv);
  // rows (queries x heads of a group) and the blocks' indices are 32-bit integers
  B3R_REQUIRE(d->Tq <= 0x7fffffff && d->Tk <= 0x7fffffff && (int64_t)d->Lq * (d->Hq / d->Hkv) <= 0x7fffff00 && d->Lk <= 0x7fffff00,
              "attention: more rows than 32-bit indices reach");
  B3R_REQUIRE((int64_t)d->B * d->Hq <= 65535, "attention: more than 65535 sequences x heads");
  return B3R_OK;
}

int attn_check(const b3r_attention_desc* d, bool backward) {
  B3R_TRY(attn_check_sizes(d));
  B3R_REQUIRE(d->scale > 0.f, "attention: the scale must be positive");
  B3R_REQUIRE((d->cu_q == nullptr) == (d->cu_k == nullptr), "attention: packed sequences need cu_q and cu_k");
  B3R_REQUIRE(!d->cu_q || (!d->q_lens && !d->k_lens), "attention: packed sequences have no q_lens or k_lens");
  const b3r_attn_tensor* ts[] = {&d->q, &d->k, &d->v, &d->o, &d->d_o, &d->dq, &d->dk, &d->dv};
  const int64_t nq = d->cu_q ? d->Tq : d->Lq, nk = d->cu_q ? d->Tk : d->Lk;
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    const bool of_k = i == 1 || i == 2 || i >= 6;
    const int64_t rows = of_k ? nk : nq, heads = of_k ? d->Hkv : d->Hq;
    if (d->B == 0 || rows == 0) continue;
    B3R_REQUIRE(ts[i]->p, "attention: NULL tensor");
    B3R_REQUIRE(((uintptr_t)ts[i]->p & 15) == 0, "attention: tensors must be 16-byte aligned");
    auto ok = [](int64_t stride, int64_t n) { return n <= 1 || (stride > 0 && stride % 8 == 0); };
    B3R_REQUIRE(ok(ts[i]->row, rows) && ok(ts[i]->head, heads) && (d->cu_q || ok(ts[i]->batch, d->B)),
                "attention: strides must be positive multiples of 8 elements");
  }
  B3R_REQUIRE(d->B == 0 || nq == 0 || d->lse.p, "attention: NULL lse");
  return B3R_OK;
}

int attn_map(CUtensorMap* map, const b3r_attn_tensor& t, int64_t rows, int heads, int batch, int D, int dtype) {
  typedef CUresult (*encode_t)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const encode_t encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<encode_t>(f);
  }();
  if (!encode) return fail(B3R_E_CUDA, "attention: the driver has no cuTensorMapEncodeTiled");
  if (rows == 0) {                     // no keys: no load is issued, the map is never read
    *map = CUtensorMap{};
    return B3R_OK;
  }
  // the stride of a dimension of one is not used, but has to be a valid one
  const int64_t row = rows > 1 ? t.row : 128, head = heads > 1 ? t.head : 128, bat = batch > 1 ? t.batch : 128;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)bat * 2};
  const cuuint32_t box[4] = {64, 128, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult rc = encode(map, dtype == B3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                             const_cast<void*>(t.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(B3R_E_CUDA, "attention: cuTensorMapEncodeTiled failed (%d)", (int)rc);
  return B3R_OK;
}

namespace {

constexpr int kWarps = 4;

template <typename T>
__device__ __forceinline__ float dot(const T* a, const T* b, int D) {
  float s = 0.f;
  for (int c = 0; c < D; c += 8) {
    const uint4 ua = *reinterpret_cast<const uint4*>(a + c), ub = *reinterpret_cast<const uint4*>(b + c);
    const T* x = reinterpret_cast<const T*>(&ua);
    const T* y = reinterpret_cast<const T*>(&ub);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += f_of(x[j]) * f_of(y[j]);
  }
  return s;
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) k_attn_dq_rows(const __grid_constant__ b3r_attention_desc d) {
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * kWarps + (threadIdx.x >> 5), h = blockIdx.y % d.Hq, b = blockIdx.y / d.Hq;
  const AttnSeq s = attn_seq(d, b);
  if (i >= (d.cu_q ? s.ql : d.Lq)) return;
  const int kv = h / (d.Hq / d.Hkv), bound = i < s.ql ? attn_bound(s, i, d.causal) : 0;
  const T* q = attn_row<const T>(d.q, b, s.q0 + i, h);
  const T* go = attn_row<const T>(d.d_o, b, s.q0 + i, h);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (bound > 0) {
    const float delta = dot(go, attn_row<const T>(d.o, b, s.q0 + i, h), d.D);
    const float lse = *attn_row<const float>(d.lse, b, s.q0 + i, h);
    for (int j0 = 0; j0 < bound; j0 += 32) {
      const int j = j0 + lane;
      float ds = 0.f;
      if (j < bound) {
        const float p = expf(d.scale * dot(q, attn_row<const T>(d.k, b, s.k0 + j, kv), d.D) - lse);
        ds = p * (dot(go, attn_row<const T>(d.v, b, s.k0 + j, kv), d.D) - delta);
      }
      for (int t = 0; t < min(32, bound - j0); ++t) {
        const float x = __shfl_sync(0xffffffffu, ds, t);
        const T* k = attn_row<const T>(d.k, b, s.k0 + j0 + t, kv);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (lane + 32 * c < d.D) acc[c] += x * f_of(k[lane + 32 * c]);
      }
    }
  }
  T* dq = attn_row<T>(d.dq, b, s.q0 + i, h);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < d.D) dq[lane + 32 * c] = t_of<T>(d.scale * acc[c]);
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) k_attn_dkv_rows(const __grid_constant__ b3r_attention_desc d) {
  const int lane = threadIdx.x & 31;
  const int j = blockIdx.x * kWarps + (threadIdx.x >> 5), kv = blockIdx.y % d.Hkv, b = blockIdx.y / d.Hkv;
  const AttnSeq s = attn_seq(d, b);
  if (j >= (d.cu_q ? s.kl : d.Lk)) return;
  const int G = d.Hq / d.Hkv;
  float ak[4] = {0.f, 0.f, 0.f, 0.f}, av[4] = {0.f, 0.f, 0.f, 0.f};
  if (j < s.kl) {
    const T* k = attn_row<const T>(d.k, b, s.k0 + j, kv);
    const T* v = attn_row<const T>(d.v, b, s.k0 + j, kv);
    const int first = d.causal ? max(0, j - (s.kl - s.ql)) : 0;   // the first query that sees key j
    for (int h = kv * G; h < kv * G + G; ++h)
      for (int i0 = first; i0 < s.ql; i0 += 32) {
        const int i = i0 + lane;
        float p = 0.f, ds = 0.f;
        if (i < s.ql) {
          const T* go = attn_row<const T>(d.d_o, b, s.q0 + i, h);
          p = expf(d.scale * dot(attn_row<const T>(d.q, b, s.q0 + i, h), k, d.D) - *attn_row<const float>(d.lse, b, s.q0 + i, h));
          ds = p * (dot(go, v, d.D) - dot(go, attn_row<const T>(d.o, b, s.q0 + i, h), d.D));
        }
        for (int t = 0; t < min(32, s.ql - i0); ++t) {
          const float pt = __shfl_sync(0xffffffffu, p, t), dt = __shfl_sync(0xffffffffu, ds, t);
          const T* q = attn_row<const T>(d.q, b, s.q0 + i0 + t, h);
          const T* go = attn_row<const T>(d.d_o, b, s.q0 + i0 + t, h);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (lane + 32 * c < d.D) {
              av[c] += pt * f_of(go[lane + 32 * c]);
              ak[c] += dt * f_of(q[lane + 32 * c]);
            }
        }
      }
  }
  T* dk = attn_row<T>(d.dk, b, s.k0 + j, kv);
  T* dv = attn_row<T>(d.dv, b, s.k0 + j, kv);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < d.D) {
      dk[lane + 32 * c] = t_of<T>(d.scale * ak[c]);
      dv[lane + 32 * c] = t_of<T>(av[c]);
    }
}

template <typename T>
int bwd_rows(const b3r_attention_desc& d, cudaStream_t s) {
  if (d.Lq > 0) {
    k_attn_dq_rows<T><<<dim3((d.Lq + kWarps - 1) / kWarps, d.B * d.Hq), 32 * kWarps, 0, s>>>(d);
    B3R_TRY(check_launch("attention dq"));
  }
  if (d.Lk > 0) {
    k_attn_dkv_rows<T><<<dim3((d.Lk + kWarps - 1) / kWarps, d.B * d.Hkv), 32 * kWarps, 0, s>>>(d);
    B3R_TRY(check_launch("attention dk, dv"));
  }
  return B3R_OK;
}

}  // namespace
}  // namespace b3r

using namespace b3r;

extern "C" int64_t b3r_attention_bwd_work_bytes(const b3r_attention_desc* d) { return d ? 0 : -1; }

extern "C" int b3r_attention_bwd(const b3r_attention_desc* d, void* stream) {
  B3R_TRY(attn_check(d, true));
  if (d->B == 0) return B3R_OK;
  return d->dtype == B3R_BF16 ? bwd_rows<__nv_bfloat16>(*d, as_stream(stream)) : bwd_rows<__half>(*d, as_stream(stream));
}
