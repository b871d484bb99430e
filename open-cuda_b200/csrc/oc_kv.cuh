// oc_kv.cuh -- what the operators on the paged key/value cache share: the
// device view of a cache (oc_kv_cache), element conversions, the batch of
// sequences a call names, and the argument checks of the entry points.
//
// Layout: k and v are [layers][pages][kv_heads][page_size][head_dim], so one
// head's page is a contiguous [page_size][head_dim] block (attention reads a
// head at a time), one page of one layer is contiguous over the heads (page
// moves copy it whole), and page_size is a power of two (a position splits
// into page and offset by a shift).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <type_traits>

#include "oc_internal.h"
#include "oc_ptx.cuh"

namespace oc {

// Bits that kernels set in the cache's status word (oc_kv_cache.status).
enum : int {
  kKvNoPages = OC_KV_NO_PAGES,    // the pool has too few free pages
  kKvBadSeq = OC_KV_BAD_SEQUENCE, // an id outside the table, or used twice, or a child that is not empty
  kKvRowFull = OC_KV_ROW_FULL,    // a sequence would outgrow its row of the page table
  kKvBadPage = OC_KV_BAD_PAGE,    // a page number outside the pool, or a token without a page
};

struct KvView {
  void* k;
  void* v;
  int* table;
  int* seq_len;
  int* refs;
  int* status;
  int layers, pages, hk, ps_shift, d, max_seqs, max_pages;
};

inline size_t kv_esize(int dtype) { return dtype == OC_KV_F32 ? 4 : 2; }

// Checks a cache descriptor and turns it into the kernels' view.
inline int kv_view(const oc_kv_cache* c, KvView* out) {
  OC_REQUIRE(c, "kv_cache: NULL cache");
  OC_REQUIRE(c->dtype == OC_KV_F32 || c->dtype == OC_KV_F16 || c->dtype == OC_KV_BF16, "kv_cache: unknown dtype");
  OC_REQUIRE(c->k && c->v && c->page_table && c->seq_len && c->refcount && c->status, "kv_cache: NULL pointer");
  OC_REQUIRE(c->num_layers > 0 && c->num_pages > 0 && c->kv_heads > 0 && c->max_seqs > 0 && c->max_pages_per_seq > 0,
             "kv_cache: empty shape");
  OC_REQUIRE(c->head_dim > 0 && c->head_dim <= 256, "kv_cache: head_dim must be 1..256");
  OC_REQUIRE(c->page_size > 0 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
             "kv_cache: page_size must be a power of two up to 1024");
  OC_REQUIRE((int64_t)c->max_pages_per_seq * c->page_size <= INT_MAX, "kv_cache: more than 2^31 - 1 tokens in a sequence");
  const uintptr_t mis = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v);
  OC_REQUIRE(mis % kv_esize(c->dtype) == 0, "kv_cache: misaligned pool");
  int sh = 0;
  while ((1 << sh) < c->page_size) ++sh;
  *out = KvView{c->k, c->v, c->page_table, c->seq_len, c->refcount, c->status, c->num_layers, c->num_pages, c->kv_heads,
                sh, c->head_dim, c->max_seqs, c->max_pages_per_seq};
  return OC_OK;
}

// Whether n rows of wa bytes at a, sa apart, and n of wb at b, sb apart, share
// memory.  Different distances: whether the ranges do.
inline bool kv_overlap(const void* a, int64_t sa, int64_t wa, const void* b, int64_t sb, int64_t wb, int64_t n) {
  const int64_t x = (int64_t)reinterpret_cast<uintptr_t>(a), y = (int64_t)reinterpret_cast<uintptr_t>(b);
  if (x + (n - 1) * sa + wa <= y || y + (n - 1) * sb + wb <= x) return false;
  if (sa != sb) return true;
  const int64_t by = ((y - x) % sa + sa) % sa;  // from a row of a to the next row of b
  return by < wa || sa - by < wb;
}

__device__ __forceinline__ float kv_f32(float x) { return x; }
__device__ __forceinline__ float kv_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float kv_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T kv_from(float x);
template <>
__device__ __forceinline__ float kv_from<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half kv_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 kv_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// {a, b} rounded to T and packed (a in the low half).
template <typename T>
__device__ __forceinline__ uint32_t kv_pack2(float a, float b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 kv_unpack2(uint32_t x) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<__half2*>(&x));
  else
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// 16 bytes of T as floats and back.
template <typename T>
struct KvVec {
  static constexpr int N = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ void kv_unpack16(const uint4& u, float (&f)[KvVec<T>::N]) {
  const T* p = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < KvVec<T>::N; ++i) f[i] = kv_f32(p[i]);
}
template <typename T>
__device__ __forceinline__ uint4 kv_pack16(const float (&f)[KvVec<T>::N]) {
  uint4 u;
  T* p = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < KvVec<T>::N; ++i) p[i] = kv_from<T>(f[i]);
  return u;
}

// One call's list of sequences: the new tokens of entry b are rows
// [cu[b], cu[b + 1]) of the token tensors (cu NULL: row b), its sequence is
// seqs[b] (seqs NULL: b).
struct KvBatch {
  const int* cu;
  const int* seqs;
  int n, total;
};

struct KvSeq {
  int s;    // row of the page table, -1 when the id is outside it
  int len;  // tokens held, the new ones included
  int q0, nq;
};

// Ids and offsets are data of the caller: whatever they hold, the result
// stays inside the token tensors and the page table.
__device__ __forceinline__ KvSeq kv_seq(const KvView& c, const KvBatch& bt, int b) {
  KvSeq r;
  r.s = bt.seqs ? bt.seqs[b] : b;
  int q0 = bt.cu ? bt.cu[b] : b, q1 = bt.cu ? bt.cu[b + 1] : b + 1;
  q0 = min(max(q0, 0), bt.total);
  q1 = min(max(q1, q0), bt.total);
  r.q0 = q0;
  r.nq = q1 - q0;
  if (r.s < 0 || r.s >= c.max_seqs) {
    r.s = -1;
    r.len = 0;
  } else {
    r.len = min(max(c.seq_len[r.s], 0), c.max_pages << c.ps_shift);
  }
  return r;
}

// Exclusive prefix sum over the block; *total gets the sum.  warp_sums: 33
// values of shared memory.  Every thread of the block takes part.
template <typename T>
__device__ __forceinline__ T block_exclusive(T x, T* warp_sums, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  T inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();  // warp_sums of the previous call have been read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    T s = lane < warps ? warp_sums[lane] : T(0);
    T si = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, si, o);
      if (lane >= o) si += y;
    }
    warp_sums[lane] = si - s;
    if (lane == 31) warp_sums[32] = si;
  }
  __syncthreads();
  *total = warp_sums[32];
  return inc - x + warp_sums[warp];
}

}  // namespace oc
