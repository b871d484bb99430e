// oc_kv_rows.cuh -- attention over the paged cache for a few query rows per
// sequence on the CUDA cores: any type, head_dim up to 256, any alignment.
//
// Decode reads each key and value once and does 4 flops per element and query
// row: every warp streams its own 16-key tiles through its own cp.async ring
// (no block barrier while it streams), and the rows of one kv head share what
// it read.  Half a warp takes a key: each lane holds
// DP / 16 features of up to ROWS query rows and of their outputs in
// registers, the products are summed over the 16 lanes by shuffles, and each
// half warp keeps a softmax of its own (running maximum and sum, log2 units),
// four keys at a time.  The halves and warps meet in shared memory at the end
// of an item.  A key that a row does not see is left out by a predicate, not
// by a zero weight, so what it holds cannot reach the row.  Sums of values
// near the type's largest may overflow: rows that do are computed again
// (kv_row_exact).
//
// Bound: at 128 f32 features three stages of four warps take an SM's shared
// memory, so each scheduler has one warp, and waits for its chain (a dot, four
// shuffles a key and row, the softmax, the product with V): 1 token over 20000
// keys, 32 heads over 8, 72 us where the bytes need 25; 25 % of the issue
// slots, 27 % of the memory's rate.  With 64 features and one row a kv head
// two CTAs fit: 16 sequences of 4000 keys, 12 heads, 76 us = 5.2 TB/s.
#pragma once
#include "oc_kv_plan.cuh"

namespace oc {

__device__ __forceinline__ void cp_async16_zfill(void* dst, const void* src, bool there) {
  const int n = there ? 16 : 0;  // the rest of the 16 bytes is written as zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's 16-key tiles in shared memory: rows of DP elements and 16 bytes
// more (an odd number of 16-byte chunks, so that the rows' chunks spread over
// the banks).
template <typename T, int DP>
struct KvTile16 {
  static constexpr int RB = DP * (int)sizeof(T) + 16;
  static constexpr int BYTES = 16 * RB;
  static constexpr int CHUNKS = DP * (int)sizeof(T) / 16;
  static constexpr int GS = CHUNKS > 16 ? 32 : CHUNKS > 8 ? 16 : CHUNKS > 4 ? 8 : 4;  // lanes per row
  static constexpr int RS = 32 / GS;                                                  // rows per step
};

// Of key `key` (the lane's): elements from the layer's start to its row of
// the pools, -1 for a key outside [lo, hi) or on a bad page.
__device__ __forceinline__ int64_t kv_row_off(const KvAttn& a, int seq, int h, int key, int lo, int hi) {
  if (key < lo || key >= hi) return -1;
  const KvView& c = a.c;
  const int page = c.table[(size_t)seq * c.max_pages + (key >> c.ps_shift)];
  if (page < 0 || page >= c.pages) {
    atomicOr(c.status, kKvBadPage);
    return -1;
  }
  return ((((int64_t)page * c.hk + h) << c.ps_shift) + (key & ((1 << c.ps_shift) - 1))) * c.d;
}

// A result that is not finite, or that rounding to T would make infinite
// (half a step above T's largest value).
template <typename T>
__device__ __forceinline__ bool kv_lost(float y) {
  if constexpr (std::is_same<T, __half>::value) return !(fabsf(y) < 65520.0f);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return !(fabsf(y) < __uint_as_float(0x7f7f8000u));
  return !isfinite(y);
}

// Requests the 16 rows whose offsets lanes 0..15 (and 16..31 again) hold.
template <typename T, int DP>
__device__ __forceinline__ void kv_load_tile(const KvAttn& a, const T* kb, const T* vb, int64_t off, uint8_t* sk,
                                             uint8_t* sv, int lane) {
  using L = KvTile16<T, DP>;
  const int d = a.c.d;
  if (a.vec) {
    const int chunks = d * (int)sizeof(T) / 16;
#pragma unroll
    for (int s = 0; s < 16 / L::RS; ++s) {
      const int row = s * L::RS + lane / L::GS;
      const int64_t o = __shfl_sync(0xffffffffu, off, row);
      const T* ks = kb + (o < 0 ? 0 : o);
      const T* vs = vb + (o < 0 ? 0 : o);
#pragma unroll
      for (int c0 = 0; c0 < L::CHUNKS; c0 += L::GS) {
        const int ch = c0 + lane % L::GS;
        if (ch < chunks) {
          const int e = ch * (16 / (int)sizeof(T));
          cp_async16_zfill(sk + row * L::RB + ch * 16, ks + e, o >= 0);
          cp_async16_zfill(sv + row * L::RB + ch * 16, vs + e, o >= 0);
        }
      }
    }
  } else {
    for (int row = 0; row < 16; ++row) {
      const int64_t o = __shfl_sync(0xffffffffu, off, row);
      T* dk = reinterpret_cast<T*>(sk + row * L::RB);
      T* dv = reinterpret_cast<T*>(sv + row * L::RB);
      for (int e = lane; e < d; e += 32) {
        dk[e] = o >= 0 ? kb[o + e] : kv_from<T>(0.0f);
        dv[e] = o >= 0 ? vb[o + e] : kv_from<T>(0.0f);
      }
    }
  }
}

template <typename T_, int DP_, int ROWS_>
struct KvRows {
  using T = T_;
  static constexpr int DP = DP_, ROWS = ROWS_;
  using L = KvTile16<T, DP>;
  // three stages a warp; rows of 1 KB leave room for two warps
  static constexpr int WARPS = DP * (int)sizeof(T) > 512 ? 2 : 4;
  static constexpr int NS = 3;
  static constexpr int THREADS = 32 * WARPS, BK = 16 * WARPS;
  static constexpr int STAGE = 2 * L::BYTES;
  static constexpr int RING = NS * STAGE;
  static constexpr int PARTS = 2 * WARPS;  // half warps
  static constexpr int VN = 16 / (int)sizeof(T);
  static constexpr int NV = (L::CHUNKS + 15) / 16;  // 16-byte chunks of a row per lane
  static constexpr int F = NV * VN;                 // features per lane
  static constexpr size_t SMEM = (size_t)WARPS * RING;
  static constexpr int FIT = (int)(224 * 1024 / (SMEM + 1024)), CTAS = FIT < 3 ? FIT : 3;  // an SM: what shared memory and registers allow
  static_assert(PARTS * ROWS * DP * 4 <= WARPS * RING, "the partial outputs take the rings' place");
  static_assert(SMEM <= 226 * 1024, "shared memory");
};

template <typename K>
__global__ void __launch_bounds__(K::THREADS, K::CTAS) kv_rows_kernel(const __grid_constant__ KvAttn a) {
  using T = typename K::T;
  using L = typename K::L;
  constexpr int ROWS = K::ROWS, F = K::F, NV = K::NV, VN = K::VN, NS = K::NS, DP = K::DP;
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ KvPlanShared plan;
  __shared__ float pm[K::PARTS][ROWS], pl[K::PARTS][ROWS];
  pdl_wait();
  pdl_launch();
  const KvView& c = a.c;
  const int d = c.d, g = a.p.group;
  KvCursor cur;
  int64_t chunk;
  const int64_t total = plan_locate(a.p, c, a.bt, blockIdx.x, &plan, &chunk, cur);
  if (threadIdx.x == 0) plan_no_cut(a);
  if (total == 0) return;
  const int64_t u0 = chunk * blockIdx.x;
  int64_t left = min(chunk, total - u0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hw = lane >> 4, l16 = lane & 15;
  uint8_t* ring = sm + warp * K::RING;
  // what lies behind head_dim stays zero in every stage: the vector reads below take whole rows
  auto zero_tails = [&]() {
    if (d * (int)sizeof(T) < L::RB - 16)
      for (int i = lane; i < NS * 32; i += 32)
        for (int e = d; e < DP; ++e) reinterpret_cast<T*>(ring + i * L::RB)[e] = kv_from<T>(0.0f);
  };
  const T* kb = static_cast<const T*>(c.k) + a.layer_off;
  const T* vb = static_cast<const T*>(c.v) + a.layer_off;

  while (left > 0) {
    const KvItem& it = cur.it;
    const int t0 = cur.at, t1 = (int)min((int64_t)it.units, t0 + left);
    const bool whole = t0 == 0 && t1 == it.units;
    zero_tails();
    __syncwarp();
    // query rows of this lane's half: features (l16 + 16 i) * VN ..
    float q[ROWS][F], o[ROWS][F], m[ROWS], l[ROWS];
    int lo[ROWS], hi[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
      lo[r] = hi[r] = 0;
      const bool live = r < it.rows;
      const int rr = it.r0 + r;
      if (live) plan_row_range(a.p, cur.s, rr, lo[r], hi[r]);
      const T* src = static_cast<const T*>(a.q) + (int64_t)(cur.s.q0 + plan_token(a.p, rr)) * a.qs + (int64_t)(cur.h * g + rr - plan_token(a.p, rr) * g) * d;
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int e = (l16 + 16 * (i / VN)) * VN + i % VN;
        q[r][i] = live && e < d ? kv_f32(src[e]) : 0.0f;
        o[r][i] = 0.0f;
      }
    }
    // tiles of 16 keys: warp w has numbers w, w + WARPS, ... of the run
    const int ntile = t1 - t0;
    const int key0 = (it.tile0 + t0) * K::BK + warp * 16 + l16;
    auto offset = [&](int i) { return i < ntile ? kv_row_off(a, cur.s.s, cur.h, key0 + i * K::BK, it.lo, it.hi) : -1; };
    int64_t ahead_off[NS];  // the page table is asked for the first tiles at once
#pragma unroll
    for (int s = 0; s < NS; ++s) ahead_off[s] = offset(s);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
      if (s < ntile) kv_load_tile<T, DP>(a, kb, vb, ahead_off[s], ring + s * K::STAGE, ring + s * K::STAGE + L::BYTES, lane);
      cp_async_commit();
    }
    int64_t next = ahead_off[NS - 1];
    for (int i = 0; i < ntile; ++i) {
      cp_async_wait<NS - 2>();
      __syncwarp();
      const int j = i + NS - 1;
      if (j < ntile) {
        uint8_t* st = ring + (j % NS) * K::STAGE;
        kv_load_tile<T, DP>(a, kb, vb, next, st, st + L::BYTES, lane);
        next = offset(j + 1);
      }
      cp_async_commit();
      const uint8_t* sk = ring + (i % NS) * K::STAGE;
      const uint8_t* sv = sk + L::BYTES;
      const int kbase = (it.tile0 + t0 + i) * K::BK + warp * 16 + hw;
      // (unrolled, the two halves are 20 KB of code at 4 rows of 128 f32
      // features, which the warps, each at its own place, wait for: 1 token over
      // 20000 keys, 32 heads over 8, 72 us against 76 to 83 with the placement)
#pragma unroll 1
      for (int k0 = 0; k0 < 16; k0 += 8) {
        float s[4][ROWS];
        uint32_t seen[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint8_t* row = sk + (k0 + 2 * kk + hw) * L::RB;
          float x[F];
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            if (L::CHUNKS % 16 == 0 || l16 + 16 * v < L::CHUNKS) {
              kv_unpack16<T>(*reinterpret_cast<const uint4*>(row + (l16 + 16 * v) * 16),
                             *reinterpret_cast<float(*)[VN]>(x + v * VN));
            } else {
#pragma unroll
              for (int e = 0; e < VN; ++e) x[v * VN + e] = 0.0f;
            }
          }
          const int key = kbase + k0 + 2 * kk;
          seen[kk] = 0;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            float dot = 0.0f;
#pragma unroll
            for (int e = 0; e < F; ++e) dot = fmaf(q[r][e], x[e], dot);
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
            const bool vis = key >= lo[r] && key < hi[r];
            seen[kk] |= (vis ? 1u : 0u) << r;
            s[kk][r] = vis ? dot * a.scale2 : -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float mx = fmaxf(fmaxf(s[0][r], s[1][r]), fmaxf(s[2][r], s[3][r]));
          const float mn = fmaxf(m[r], mx), base = mn == -INFINITY ? 0.0f : mn;
          const float corr = exp2f(m[r] - base);
          m[r] = mn;
          float add = 0.0f;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            s[kk][r] = exp2f(s[kk][r] - base);
            add += s[kk][r];
          }
          l[r] = fmaf(l[r], corr, add);
          if (corr != 1.0f)
#pragma unroll
            for (int e = 0; e < F; ++e) o[r][e] *= corr;
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if (seen[kk] == 0) continue;
          const uint8_t* row = sv + (k0 + 2 * kk + hw) * L::RB;
          float x[F];
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            if (L::CHUNKS % 16 == 0 || l16 + 16 * v < L::CHUNKS) {
              kv_unpack16<T>(*reinterpret_cast<const uint4*>(row + (l16 + 16 * v) * 16),
                             *reinterpret_cast<float(*)[VN]>(x + v * VN));
            } else {
#pragma unroll
              for (int e = 0; e < VN; ++e) x[v * VN + e] = 0.0f;
            }
          }
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            if ((seen[kk] >> r) & 1u)
#pragma unroll
              for (int e = 0; e < F; ++e) o[r][e] = fmaf(s[kk][r], x[e], o[r][e]);
        }
        __syncwarp();  // the halves may have parted at a skipped key
      }
    }
    // the half warps meet: partial outputs in the rings' place
    cp_async_wait<0>();
    __syncthreads();
    float* po = reinterpret_cast<float*>(sm);  // [PARTS][ROWS][DP]
    const int part = warp * 2 + hw;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (l16 == 0) pm[part][r] = m[r], pl[part][r] = l[r];
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int e = (l16 + 16 * (i / VN)) * VN + i % VN;
        if (e < DP) po[(part * ROWS + r) * DP + e] = o[r][i];
      }
    }
    __syncthreads();
    float* slot = whole ? nullptr : plan_slot(a, blockIdx.x, t0 == 0 ? 1 : 0, DP);
    bool lost = false;  // a result of this thread's is not finite
    for (int x = threadIdx.x; x < it.rows * DP; x += K::THREADS) {
      const int r = x / DP, e = x % DP;
      float mm = pm[0][r];
#pragma unroll
      for (int k = 1; k < K::PARTS; ++k) mm = fmaxf(mm, pm[k][r]);
      const float base = mm == -INFINITY ? 0.0f : mm;
      float ls = 0.0f, os = 0.0f;
#pragma unroll
      for (int k = 0; k < K::PARTS; ++k) {
        const float w = exp2f(pm[k][r] - base);
        ls = fmaf(w, pl[k][r], ls);
        os = fmaf(w, po[(k * ROWS + r) * DP + e], os);
      }
      if (whole) {
        const int rr = it.r0 + r;
        if (e < d) {
          const float y = ls == 0.0f ? 0.0f : os / ls;
          static_cast<T*>(a.out)[(int64_t)(cur.s.q0 + plan_token(a.p, rr)) * a.os + (int64_t)(cur.h * g + rr - plan_token(a.p, rr) * g) * d + e] =
              kv_from<T>(y);
          lost |= kv_lost<T>(y);
        }
      } else {
        if (e == 0) slot[r] = mm, slot[ROWS + r] = ls;
        slot[plan_slot_o(ROWS) + (size_t)r * DP + e] = os;
      }
    }
    if (__syncthreads_or(lost) && threadIdx.x == 0) plan_lost(a);
    if (t0 == 0 && !whole && threadIdx.x == 0) plan_cut(a, cur, it.units - t1, chunk);
    left -= t1 - t0;
    if (left > 0) plan_next(a.p, c, a.bt, cur);
  }
}

}  // namespace oc
