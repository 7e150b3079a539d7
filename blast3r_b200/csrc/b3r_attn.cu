// Part 5 of the C ABI, attention: what both passes check, the tensor maps that they load by, and the packed rows
// that they do not reach.
#include <algorithm>
#include <cmath>
#include <utility>
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
  B3R_REQUIRE((int64_t)d->B * d->Hq <= 0x7fffffff, "attention: too many sequences x heads");
  return B3R_OK;
}

int attn_check(const b3r_attention_desc* d, bool backward) {
  B3R_TRY(attn_check_sizes(d));
  // (from 2^-100 on the backward pass's lse / scale is a float32 too)
  B3R_REQUIRE(d->scale >= 0x1p-100f && d->scale < INFINITY, "attention: the scale must be positive and finite, 2^-100 at least");
  B3R_REQUIRE((d->cu_q == nullptr) == (d->cu_k == nullptr), "attention: packed sequences need cu_q and cu_k");
  B3R_REQUIRE(!d->cu_q || (!d->q_lens && !d->k_lens), "attention: packed sequences have no q_lens or k_lens");
  const b3r_attn_tensor* ts[] = {&d->q, &d->k, &d->v, &d->o, &d->d_o, &d->dq, &d->dk, &d->dv};
  const int64_t nq = d->cu_q ? d->Tq : d->Lq, nk = d->cu_q ? d->Tk : d->Lk;
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    const bool of_k = i == 1 || i == 2 || i >= 6;
    const int64_t rows = of_k ? nk : nq, heads = of_k ? d->Hkv : d->Hq;
    if ((d->B == 0 && !d->cu_q) || rows == 0) continue;
    B3R_REQUIRE(ts[i]->p, "attention: NULL tensor");
    B3R_REQUIRE(((uintptr_t)ts[i]->p & 15) == 0, "attention: tensors must be 16-byte aligned");
    auto ok = [](int64_t stride, int64_t n) { return n <= 1 || (stride > 0 && stride % 8 == 0); };
    B3R_REQUIRE(ok(ts[i]->row, rows) && ok(ts[i]->head, heads) && (d->cu_q || ok(ts[i]->batch, d->B)),
                "attention: strides must be positive multiples of 8 elements");
  }
  B3R_REQUIRE((d->B == 0 && !d->cu_q) || nq == 0 || d->lse.p, "attention: NULL lse");
  return B3R_OK;
}

static int encode_map(CUtensorMap* map, const b3r_attn_tensor& t, int64_t rows, int heads, int G, int batch, int D, int dtype, int box_rows) {
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
  // the encoder wants a current context, which a thread that has made no runtime call yet (an
  // autograd worker) does not have
  static thread_local int ready = -1;
  int dev;
  B3R_TRY(check_cuda(cudaGetDevice(&dev), "attention"));
  if (dev != ready) {
    B3R_TRY(check_cuda(cudaSetDevice(dev), "attention"));
    ready = dev;
  }
  if (!encode) return fail(B3R_E_CUDA, "attention: the driver has no cuTensorMapEncodeTiled");
  if (rows == 0) {                     // no keys: no load is issued, the map is never read
    *map = CUtensorMap{};
    return B3R_OK;
  }
  // the stride of a dimension of one is not used, but has to be a valid one
  const int64_t row = rows > 1 ? t.row : 128, head = heads > 1 ? t.head : 128, bat = batch > 1 ? t.batch : 128;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
  cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)bat * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  if (G > 0) {                         // heads before rows
    std::swap(dims[1], dims[2]);
    std::swap(strides[0], strides[1]);
    box[1] = (cuuint32_t)G;
    box[2] = (cuuint32_t)(box_rows / G);
  }
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult rc = encode(map, dtype == B3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                             const_cast<void*>(t.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(B3R_E_CUDA, "attention: cuTensorMapEncodeTiled failed (%d)", (int)rc);
  return B3R_OK;
}

// Packed rows of no sequence: before the first, past the last, or past the bounds Lq / Lk of a length.  A thread looks
// one row up among the offsets, and its warp clears those that were found outside.  Nothing to clear is the usual
// case, and takes a launch's latency (2.2 us for 13 thousand rows in 20 sequences on one B200).
namespace {
constexpr int kClearRows = 128;
__global__ void __launch_bounds__(kClearRows) k_attn_clear(const __grid_constant__ b3r_attention_desc d, int backward) {
  const bool of_k = blockIdx.y == 1;
  const int32_t* cu = of_k ? d.cu_k : d.cu_q;
  const int64_t T = of_k ? d.Tk : d.Tq, row = (int64_t)blockIdx.x * kClearRows + threadIdx.x;
  const int lane = threadIdx.x & 31, most = of_k ? d.Lk : d.Lq, heads = of_k ? d.Hkv : d.Hq, chunks = d.D / 8;
  bool off = false;
  if (row < T) {
    int lo = 0, hi = d.B + 1;                          // offsets up to this row: those before lo, and none from hi on
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (cu[mid] <= row) lo = mid + 1;
      else hi = mid;
    }
    off = lo == 0 || lo > d.B || row - max(cu[lo - 1], 0) >= most;
  }
  for (uint32_t left = __ballot_sync(0xffffffffu, off); left; left &= left - 1) {
    const int64_t r = row - lane + __ffs(left) - 1;
    for (int i = lane; i < heads * chunks; i += 32) {
      const int h = i / chunks, c = (i - h * chunks) * 8;
      auto zero = [&](const b3r_attn_tensor& t) { *reinterpret_cast<uint4*>(attn_row<uint16_t>(t, 0, r, h) + c) = make_uint4(0, 0, 0, 0); };
      if (!backward) {
        zero(d.o);
        if (c == 0) *attn_row<float>(d.lse, 0, r, h) = -INFINITY;
      } else if (!of_k) {
        zero(d.dq);
      } else {
        zero(d.dk);
        zero(d.dv);
      }
    }
  }
}
}  // namespace

int attn_clear(const b3r_attention_desc* d, bool backward, cudaStream_t s) {
  const int64_t rows = backward ? std::max(d->Tq, d->Tk) : d->Tq;
  if (!d->cu_q || rows == 0) return B3R_OK;
  k_attn_clear<<<dim3((unsigned)((rows + kClearRows - 1) / kClearRows), backward ? 2 : 1), kClearRows, 0, s>>>(*d, backward);
  return check_launch("attention");
}

int attn_map(CUtensorMap* map, const b3r_attn_tensor& t, int64_t rows, int heads, int batch, int D, int dtype, int box) {
  return encode_map(map, t, rows, heads, 0, batch, D, dtype, box);
}
int attn_map_groups(CUtensorMap* map, const b3r_attn_tensor& t, int64_t rows, int heads, int G, int batch, int D, int dtype) {
  return encode_map(map, t, rows, heads, G, batch, D, dtype, 128);
}

}  // namespace b3r
