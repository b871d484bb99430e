// oc_kv_mma.cuh -- attention over the paged cache in items of 16 query rows,
// f16 and bf16: decode steps, and chunks that the tcgen05 tiles do not take
// (head_dims over 128; items of 32 rows: queries that are not 16-byte aligned).
//
// Bound: the cache's bytes (a decode step of 8 rows does 32 flops per element
// read).  On the CUDA cores 8 rows cost more issue slots than the memory
// leaves (0.1 of the copy rate measured, 3.7 ms for 64 sequences of 2 to 15 k
// keys, 32 heads of 128 over 8; here 387 to 405 us a call among others = 5.6 to
// 5.8 TB/s, 0.87 to 0.9), so the products run on warp-level matrix instructions, whose 16 rows a decode
// step's query heads of one kv head fill in part; tcgen05 tiles of 128 rows
// would be mostly empty and would put a block-wide hand-over behind every
// tile.  A warp works alone: its own 16-key tiles, its own cp.async ring, its
// own softmax; only the end of an item is a meeting.
//   S = Q K^T   16 rows x 16 keys: two m16n8k16 per 16 features (K read with
//               ldmatrix: its rows are the columns of the second operand)
//   O += P V    two m16n8k16 per 16 features (V read with ldmatrix.trans),
//               once with P rounded to the type and once with what the
//               rounding left (p - round(p)), so that the weights carry 16 or
//               more bits (f16: from 2^-24 of the row's largest on, 2^-40 of
//               it below): the memory-bound kernel has the issue slots, and
//               the result then differs from f32 arithmetic by less than its
//               own last rounding
// A weight of a key that a row does not see is 0, but 0 times an infinity or
// NaN is NaN: a row whose result is not finite is computed again
// (kv_row_exact), so that what it does not see has no part in it.
#pragma once
#include "oc_kv_rows.cuh"

namespace oc {

__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d (16 x 8, f32) += a (16 x 16) b (16 x 8)
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T_, int DP_, int MT_>
struct KvMma {
  using T = T_;
  static constexpr int DP = DP_, MT = MT_, ROWS = 16 * MT;
  using L = KvTile16<T, DP>;
  static constexpr int WARPS = 4, THREADS = 32 * WARPS, BK = 16 * WARPS;
  // stages and CTAs an SM: the warps hide one another's latencies better than
  // more stages do (64 sequences, 2.26 GB of cache, 16 rows of 128 features:
  // 3 x 2 stages 386 us, 2 x 3 stages 416)
  static constexpr int NS = DP <= 64 ? 4 : DP <= 128 && MT == 1 ? 2 : 3;
  static constexpr int CTAS = DP <= 64 ? 3 : DP > 128 ? 1 : MT == 1 ? 3 : 2;
  static constexpr int STAGE = 2 * L::BYTES, RING = NS * STAGE;
  static constexpr int OS = DP + 8;                       // floats of a row of partial outputs
  static constexpr bool QREG = DP <= 128 && MT == 1;      // query fragments stay in registers
  // f16 weights times 2^15, so that 2^-39 of the largest is still half a step
  // of f16 (at 1 it would be 2^-25, and 2^17 keys of that make 2^-8)
  static constexpr float P_UNIT = std::is_same<T, __half>::value ? 32768.0f : 1.0f;
  static constexpr size_t SMEM = (size_t)WARPS * RING + ROWS * L::RB;
  static_assert(WARPS * ROWS * OS * 4 <= WARPS * RING, "the partial outputs take the rings' place");
  static_assert(SMEM <= 226 * 1024, "shared memory");
};

template <typename K>
__global__ void __launch_bounds__(K::THREADS, K::CTAS) kv_mma_kernel(const __grid_constant__ KvAttn a) {
  using T = typename K::T;
  using L = typename K::L;
  constexpr int DP = K::DP, MT = K::MT, NS = K::NS, KS = DP / 16, ROWS = K::ROWS, OS = K::OS;
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ KvPlanShared plan;
  __shared__ float pm[K::WARPS][ROWS], pl[K::WARPS][ROWS];
  pdl_wait();
  pdl_launch();
  const KvView& c = a.c;
  const int d = c.d, g = a.p.group;
  KvCursor cur;
  int64_t chunk;
  const int64_t total = plan_locate(a.p, c, a.bt, blockIdx.x, &plan, &chunk, cur);
  if (threadIdx.x == 0) plan_no_cut(a);
  if (total == 0) return;
  int64_t left = min(chunk, total - chunk * blockIdx.x);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = sm + warp * K::RING;
  uint8_t* sq = sm + K::WARPS * K::RING;
  const T* kb = static_cast<const T*>(c.k) + a.layer_off;
  const T* vb = static_cast<const T*>(c.v) + a.layer_off;
  // ldmatrix addresses of this lane within a tile: K has keys 0-7 / 8-15 in
  // lanes 0-15 / 16-31 and the two halves of 16 features alternating every 8;
  // V (transposed) the halves of the features in lanes 0-15 / 16-31 and keys
  // 0-7 / 8-15 alternating
  const uint32_t k_off = (uint32_t)(((lane >> 4) * 8 + (lane & 7)) * L::RB + ((lane >> 3) & 1) * 16);
  const uint32_t v_off = (uint32_t)((((lane >> 3) & 1) * 8 + (lane & 7)) * L::RB + (lane >> 4) * 16);
  const uint32_t q_off = (uint32_t)((lane & 15) * L::RB + (lane >> 4) * 16);

  while (left > 0) {
    const KvItem& it = cur.it;
    const int t0 = cur.at, t1 = (int)min((int64_t)it.units, t0 + left);
    const bool whole = t0 == 0 && t1 == it.units;
    if (d < DP) {  // what lies behind head_dim is zero in every stage
      for (int i = lane; i < NS * 32; i += 32)
        for (int e = d; e < DP; e += 8) *reinterpret_cast<uint4*>(ring + i * L::RB + e * 2) = make_uint4(0, 0, 0, 0);
    }
    // the first tiles are on their way while the queries are fetched
    const int ntile = t1 - t0;
    const int key0 = (it.tile0 + t0) * K::BK + warp * 16;
    auto offset = [&](int i) {
      return i < ntile ? kv_row_off(a, cur.s.s, cur.h, key0 + (lane & 15) + i * K::BK, it.lo, it.hi) : -1;
    };
    int64_t ahead_off[NS];  // the page table is asked for the first tiles at once
#pragma unroll
    for (int s = 0; s < NS; ++s) ahead_off[s] = offset(s);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
      if (s < ntile) kv_load_tile<T, DP>(a, kb, vb, ahead_off[s], ring + s * K::STAGE, ring + s * K::STAGE + L::BYTES, lane);
      cp_async_commit();
    }
    int64_t next = ahead_off[NS - 1];
    if (a.qvec) {
      for (int x = threadIdx.x; x < ROWS * (DP / 8); x += K::THREADS) {
        const int r = x / (DP / 8), e = x % (DP / 8) * 8, rr = it.r0 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < it.rows && e < d)
          v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(cur.s.q0 + plan_token(a.p, rr)) * a.qs +
                                              (int64_t)(cur.h * g + rr - plan_token(a.p, rr) * g) * d + e);
        *reinterpret_cast<uint4*>(sq + r * L::RB + e * 2) = v;
      }
    } else {
      for (int x = threadIdx.x; x < ROWS * DP; x += K::THREADS) {
        const int r = x / DP, e = x % DP, rr = it.r0 + r;
        T v = kv_from<T>(0.0f);
        if (r < it.rows && e < d)
          v = static_cast<const T*>(a.q)[(int64_t)(cur.s.q0 + plan_token(a.p, rr)) * a.qs + (int64_t)(cur.h * g + rr - plan_token(a.p, rr) * g) * d + e];
        *reinterpret_cast<T*>(sq + r * L::RB + e * 2) = v;
      }
    }
    __syncthreads();
    // rows of this lane: (lane / 4) and that + 8 of each 16; what they see
    int lo[MT][2], hi[MT][2];
    float o[MT][DP / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = t * 16 + i * 8 + (lane >> 2);
        lo[t][i] = hi[t][i] = 0;
        if (r < it.rows) plan_row_range(a.p, cur.s, it.r0 + r, lo[t][i], hi[t][i]);
        m[t][i] = -INFINITY, l[t][i] = 0.0f;
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][n][i] = 0.0f;
    }
    // keys that every row of the item sees: [all_lo, all_hi)
    int all_lo, all_hi, unused;
    plan_row_range(a.p, cur.s, it.r0, unused, all_hi);
    plan_row_range(a.p, cur.s, it.r0 + it.rows - 1, all_lo, unused);
    uint32_t qf[K::QREG ? KS : 1][4];
    if constexpr (K::QREG) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) ldsm4(qf[ks], smem_u32(sq) + q_off + ks * 32);
    }
    for (int i = 0; i < ntile; ++i) {
      cp_async_wait<NS - 2>();
      __syncwarp();
      const int ahead = i + NS - 1;
      if (ahead < ntile) {
        uint8_t* st = ring + (ahead % NS) * K::STAGE;
        kv_load_tile<T, DP>(a, kb, vb, next, st, st + L::BYTES, lane);
        next = offset(ahead + 1);
      }
      cp_async_commit();
      const uint32_t sk = smem_u32(ring + (i % NS) * K::STAGE), sv = sk + L::BYTES;
      const int base = key0 + i * K::BK;
      float s[MT][2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][n][e] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t b[4];
        ldsm4(b, sk + k_off + ks * 32);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if constexpr (K::QREG) {
            mma16816<T>(s[t][0], qf[ks], b[0], b[1]);
            mma16816<T>(s[t][1], qf[ks], b[2], b[3]);
          } else {
            uint32_t af[4];
            ldsm4(af, smem_u32(sq) + t * 16 * L::RB + q_off + ks * 32);
            mma16816<T>(s[t][0], af, b[0], b[1]);
            mma16816<T>(s[t][1], af, b[2], b[3]);
          }
        }
      }
      const bool free_of_masks = base >= all_lo && base + 16 <= all_hi;
      uint32_t ph[MT][4], pr[MT][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = base + n * 8 + (lane & 3) * 2 + (e & 1);
            const float x = s[t][n][e] * a.scale2;
            s[t][n][e] = free_of_masks || (key >= lo[t][e >> 1] && key < hi[t][e >> 1]) ? x : -INFINITY;
          }
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          float mx = fmaxf(fmaxf(s[t][0][2 * i2], s[t][0][2 * i2 + 1]), fmaxf(s[t][1][2 * i2], s[t][1][2 * i2 + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[t][i2], mx), bs = mn == -INFINITY ? 0.0f : mn;
          const float corr = kv_ex2(m[t][i2] - bs);
          m[t][i2] = mn;
          float add = 0.0f;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float p = kv_ex2(s[t][n][2 * i2 + e] - bs) * K::P_UNIT;
              s[t][n][2 * i2 + e] = p;
              add += p;
            }
          l[t][i2] = fmaf(l[t][i2], corr, add);
          if (__any_sync(0xffffffffu, corr != 1.0f)) {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              o[t][n][2 * i2] *= corr;
              o[t][n][2 * i2 + 1] *= corr;
            }
          }
        }
        // the accumulator layout of S is the operand layout of P
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            const float p0 = s[t][n][2 * i2], p1 = s[t][n][2 * i2 + 1];
            const uint32_t hp = kv_pack2<T>(p0, p1);
            const float2 back = kv_unpack2<T>(hp);
            ph[t][2 * n + i2] = hp;
            pr[t][2 * n + i2] = kv_pack2<T>(p0 - back.x, p1 - back.y);
          }
      }
#pragma unroll
      for (int n = 0; n < KS; ++n) {
        uint32_t b[4];
        ldsm4_t(b, sv + v_off + n * 32);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          mma16816<T>(o[t][2 * n], ph[t], b[0], b[1]);
          mma16816<T>(o[t][2 * n + 1], ph[t], b[2], b[3]);
          mma16816<T>(o[t][2 * n], pr[t], b[0], b[1]);
          mma16816<T>(o[t][2 * n + 1], pr[t], b[2], b[3]);
        }
      }
    }
    // the warps meet: partial outputs in the rings' place
    cp_async_wait<0>();
    __syncthreads();
    float* po = reinterpret_cast<float*>(sm);  // [WARPS][ROWS][OS]
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        const int r = t * 16 + i2 * 8 + (lane >> 2);
        float ls = l[t][i2];
        ls += __shfl_xor_sync(0xffffffffu, ls, 1);
        ls += __shfl_xor_sync(0xffffffffu, ls, 2);
        if ((lane & 3) == 0) pm[warp][r] = m[t][i2], pl[warp][r] = ls;
        float* row = po + (warp * ROWS + r) * OS + (lane & 3) * 2;
        if (r < it.rows)
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
            *reinterpret_cast<float2*>(row + n * 8) = make_float2(o[t][n][2 * i2], o[t][n][2 * i2 + 1]);
      }
    __syncthreads();
    float* slot = whole ? nullptr : plan_slot(a, blockIdx.x, t0 == 0 ? 1 : 0, DP);
    bool lost = false;  // a result of this thread's is not finite
    for (int x = threadIdx.x; x < it.rows * (DP / 2); x += K::THREADS) {
      const int r = x / (DP / 2), e = x % (DP / 2) * 2;
      float mm = pm[0][r];
#pragma unroll
      for (int k = 1; k < K::WARPS; ++k) mm = fmaxf(mm, pm[k][r]);
      const float bs = mm == -INFINITY ? 0.0f : mm;
      float ls = 0.0f;
      float2 os = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < K::WARPS; ++k) {
        const float w = kv_ex2(pm[k][r] - bs);
        const float2 y = *reinterpret_cast<const float2*>(po + (k * ROWS + r) * OS + e);
        ls = fmaf(w, pl[k][r], ls);
        os.x = fmaf(w, y.x, os.x);
        os.y = fmaf(w, y.y, os.y);
      }
      if (whole) {
        const int rr = it.r0 + r;
        if (e < d) {
          const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
          os.x *= inv, os.y *= inv;
          lost |= kv_lost<T>(os.x) || kv_lost<T>(os.y);
          T* out = static_cast<T*>(a.out) + (int64_t)(cur.s.q0 + plan_token(a.p, rr)) * a.os + (int64_t)(cur.h * g + rr - plan_token(a.p, rr) * g) * d + e;
          if (a.ovec) {
            *reinterpret_cast<uint32_t*>(out) = kv_pack2<T>(os.x, os.y);
          } else {
            out[0] = kv_from<T>(os.x);
            out[1] = kv_from<T>(os.y);
          }
        }
      } else {
        if (e == 0) slot[r] = mm, slot[ROWS + r] = ls;
        *reinterpret_cast<float2*>(slot + plan_slot_o(ROWS) + (size_t)r * DP + e) = os;
      }
    }
    if (__syncthreads_or(lost) && threadIdx.x == 0) plan_lost(a);
    if (t0 == 0 && !whole && threadIdx.x == 0) plan_cut(a, cur, it.units - t1, chunk);
    left -= t1 - t0;
    if (left > 0) plan_next(a.p, c, a.bt, cur);
  }
}

}  // namespace oc
