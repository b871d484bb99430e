// oc_kv_tile32.cuh -- attention over the paged cache for chunks of new tokens
// in f32 on the tcgen05 tensor cores (D: head_dim, or 64 or 128 above it).
//
// The arithmetic is flash_tc_kernel's (oc_flash_tc.cuh): every operand as two
// f16 terms of a power-of-two scaling (Q and K per row, V per tile, P by
// 2^15), three MMAs per product step (the small terms first), scores in log2
// units, the running output rescaled with every tile.  What differs is where rows come from and how the
// work is shared out: query rows are the heads of a kv head of consecutive
// tokens, key rows are looked up page by page (zeros where no row of the item
// sees a key), a CTA works through a run of pieces (oc_kv_plan.cuh), and what
// a cut leaves goes to the workspace.
//
// Bound: not the tensor pipe but the chain of a tile, S -> softmax (two passes
// over tensor memory) -> P V -> next S, about 8000 cycles at d = 64, and the
// conversion of K and V beside it.  Measured: 8 prompts of 300 to 777 tokens
// over contexts of 800 to 1000, 12 heads of 64: 125 us a call (63 TFLOP/s of
// visible products; the CUDA cores took 1220).  S in two buffers with K
// converted a tile ahead measured slower (167 us : 143 then: the softmax
// warps, which share their schedulers with the converters, spill).
//
// One CTA an SM, 448 threads:
//   warp 0       TMEM allocator + MMA issuer (lane 0)
//   warps 1..8   converters: f32 rows -> f16 terms in swizzled tiles
//   warps 9..12  softmax and output: thread = query row = TMEM lane
//   warp 13      walks the CTA's run and hands its pieces to the others
#pragma once
#include <cstddef>

#include "oc_kv_tile.cuh"

namespace oc {

template <int D_>
struct KvTile32 {
  static constexpr int D = D_, DP = D_, ROWS = 128, BK = 128, THREADS = 32 * 14;
  static constexpr int PANEL = 128 * 128, TILE = 128 * D * 2;  // bytes: 64 features, one term of 128 rows
  static constexpr int S_COL = 0, O_COL = 128, A_COL = 128 + D, TMEM_COLS = D == 64 ? 256 : 512;
  static constexpr size_t SMEM = 1024 + 6 * (size_t)TILE;
};

struct KvTile32Shared {
  uint64_t q_full, q_empty, k_full, k_empty, v_full, v_empty, s_full, p_full, o_full, o_empty, vmax;
  uint64_t job_full[kJobs], job_empty[kJobs];
  KvJob ring[kJobs];
  float icq[2][128];              // 1 / c_q per query row, by the piece's parity
  alignas(16) float ick[2][128];  // 1 / c_k per key row, with the sign of the scale, by the tile's parity (read four at a time)
  alignas(16) float short_of[2][128];  // by the tile's parity, per key: what V's row lacks to keep its bits (kv_convert_values)
  alignas(8) uint8_t uneven[2][8];     // by the tile's parity, per converter warp: some of its rows lack any
  float icv[2];                        // 1 / c_v of the V tile
  float vpart[2][kFaConv];             // converter warps' max |v|
  uint32_t tmem;
  int abort_word;
};
static_assert(offsetof(KvTile32Shared, ick) % 16 == 0 && alignof(KvTile32Shared) % 16 == 0 && offsetof(KvTile32Shared, short_of) % 16 == 0,
              "read as float4");
static_assert(kFaConv == 8, "a tile's `uneven` is read as one 64-bit word");

// The converter warp's 16 rows of a 128-row tile, from the offsets that its
// lanes 0..15 hold (-1: a row of zeros): float4 q4 of row s * RPS + ro in x[s].
template <int D>
struct KvConvert {
  static constexpr int RPW = 128 / kFaConv, LPR = D / 4, RPS = 32 / LPR, NS = RPW / RPS;
  static __device__ __forceinline__ void load(const float* __restrict__ base, int64_t off, int d, bool vec, int lane, float4 (&x)[NS]) {
    const int q4 = lane % LPR, ro = lane / LPR;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int64_t o = __shfl_sync(0xffffffffu, off, s * RPS + ro);
      x[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (o >= 0 && 4 * q4 < d) {
        const float* p = base + o + 4 * q4;
        const int left = d - 4 * q4;  // zeros behind head_dim
        if (vec)
          x[s] = *reinterpret_cast<const float4*>(p);
        else
          x[s] = make_float4(p[0], left > 1 ? p[1] : 0.0f, left > 2 ? p[2] : 0.0f, left > 3 ? p[3] : 0.0f);
      }
    }
  }
  static __device__ __forceinline__ void store(const float4& x, float c, int row, int q4, uint8_t* thi, uint8_t* tlo) {
    uint2 hi, lo;
    fa_split4(x, c, hi, lo);
    const uint32_t to = fa_tile_off(row, 4 * q4);
    *reinterpret_cast<uint2*>(thi + to) = hi;
    *reinterpret_cast<uint2*>(tlo + to) = lo;
  }
};

// Rows of queries or keys, each by its own power of two c; inv: sign / c.
template <int D>
__device__ __forceinline__ void kv_convert_rows(const float* __restrict__ base, int64_t off, int d, bool vec, uint8_t* thi, uint8_t* tlo,
                                                float* inv, float sign, int w, int lane) {
  using C = KvConvert<D>;
  const int q4 = lane % C::LPR, ro = lane / C::LPR;
  float4 x[C::NS];
  C::load(base, off, d, vec, lane, x);
  float mx[C::NS];
#pragma unroll
  for (int s = 0; s < C::NS; ++s) mx[s] = fa_absmax4(x[s]);
#pragma unroll
  for (int o = C::LPR / 2; o > 0; o >>= 1)
#pragma unroll
    for (int s = 0; s < C::NS; ++s) mx[s] = fmaxf(mx[s], __shfl_xor_sync(0xffffffffu, mx[s], o));
#pragma unroll
  for (int s = 0; s < C::NS; ++s) {
    const int ce = fa_range_exp(mx[s]), row = w * C::RPW + s * C::RPS + ro;
    if (q4 == 0) inv[row] = __fmul_rn(sign, exp2_int(-ce));
    C::store(x[s], exp2_int(ce), row, q4, thi, tlo);
  }
}

// Rows of values, all by one power of two c that puts the tile's largest into
// [2^14, 2^15): through `part` and the barrier `vmax`.  Two f16 terms of a
// scaled value t are off by at most 2^-24 (both in f16's subnormal steps) or
// 2^-21 |t|, so a row whose largest is r keeps 2^-22 of it only from r c = 1/4
// on.  short_of[key] = 1/4 - r c (0 for a row of zeros, which is exact), and
// uneven[w] tells the softmax to ask whether the keys it weighs fall short on
// the whole: a row of queries whose weights p have sum(p short_of) > 0 would
// lose bits, whether it does not see the large values or gives them no weight.
// Measured, 8 prompts of 300 to 777 tokens over contexts of 800 to 1000, 12
// heads of 64: 126 us; with one value row in each of 2^-10 of the others 124,
// of 2^-20 125.
template <int D>
__device__ __forceinline__ bool kv_convert_values(const float* __restrict__ base, int64_t off, int d, bool vec, uint8_t* thi, uint8_t* tlo,
                                                  float* inv, int w, int lane, float* part, uint64_t* vmax, uint32_t ph, float* short_of,
                                                  uint8_t* uneven, volatile int* abort_flag) {
  using C = KvConvert<D>;
  const int q4 = lane % C::LPR, ro = lane / C::LPR;
  float4 x[C::NS];
  C::load(base, off, d, vec, lane, x);
  // the rows' maxima: lanes that differ in bit 1 << b of q4 halve the rows
  // between them, so that lane q4 ends up with row (q4 & (NS - 1)) * RPS + ro
  float mx[C::NS];
#pragma unroll
  for (int s = 0; s < C::NS; ++s) mx[s] = fa_absmax4(x[s]);
#pragma unroll
  for (int n = C::NS / 2; n > 0; n >>= 1) {
    const bool upper = (q4 & n) != 0;
#pragma unroll
    for (int s = 0; s < n; ++s) {
      const float keep = upper ? mx[s + n] : mx[s], give = upper ? mx[s] : mx[s + n];
      mx[s] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, n));
    }
  }
#pragma unroll
  for (int o = C::NS; o < C::LPR; o <<= 1) mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
  const float row_max = mx[0];
  float m = row_max;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) {
    part[w] = m;
    mbar_arrive(vmax);
  }
  if (!warp_wait(vmax, ph, abort_flag)) return false;
  m = part[0];
#pragma unroll
  for (int j = 1; j < kFaConv; ++j) m = fmaxf(m, part[j]);
  const int ce = fa_range_exp(m);
  const float c = exp2_int(ce);
  const float lacks = row_max > 0.0f ? 0.25f - row_max * c : 0.0f;
  if (q4 < C::NS) short_of[w * C::RPW + q4 * C::RPS + ro] = lacks;
  const bool some = __any_sync(0xffffffffu, lacks > 0.0f);
  if (lane == 0) uneven[w] = some;
  if (w == 0 && lane == 0) *inv = exp2_int(-ce);
#pragma unroll
  for (int s = 0; s < C::NS; ++s) C::store(x[s], c, w * C::RPW + s * C::RPS + ro, q4, thi, tlo);
  return true;
}

// Scores outside [from, to) of a 32-key chunk become `out`.
__device__ __forceinline__ void kv_mask_chunk(uint32_t (&r)[32], int from, int to, uint32_t out) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j < from || j >= to) r[j] = out;
}

template <typename K>
__global__ void __launch_bounds__(K::THREADS, 1) kv_tile32_kernel(const __grid_constant__ KvAttn a) {
  constexpr int D = K::D;
  extern __shared__ uint8_t raw[];
  __shared__ KvPlanShared plan;
  __shared__ KvTile32Shared sh;
  volatile int* abort_flag = &sh.abort_word;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  // V precedes K: the V descriptors' reach stays inside the allocation
  uint8_t *q_hi = base, *q_lo = q_hi + K::TILE, *v_hi = q_lo + K::TILE, *v_lo = v_hi + K::TILE, *k_hi = v_lo + K::TILE,
          *k_lo = k_hi + K::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!a.beside) pdl_wait();  // (oc_kv_tile.cuh)
  pdl_launch();
  const KvView& c = a.c;
  KvCursor cur;
  int64_t chunk;
  const int64_t total = plan_locate(a.p, c, a.bt, blockIdx.x, &plan, &chunk, cur);
  if (threadIdx.x == 0) plan_no_cut(a);
  if (total == 0) {
    pdl_wait();
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, kFaConv);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.k_full, kFaConv);
    mbar_init(&sh.k_empty, 1);
    mbar_init(&sh.v_full, kFaConv);
    mbar_init(&sh.v_empty, 1);
    mbar_init(&sh.s_full, 1);
    mbar_init(&sh.p_full, 4);
    mbar_init(&sh.o_full, 1);
    mbar_init(&sh.o_empty, 4);
    mbar_init(&sh.vmax, kFaConv);
    for (int i = 0; i < kJobs; ++i) {
      mbar_init(&sh.job_full[i], 1);
      mbar_init(&sh.job_empty[i], 1 + kFaConv + 4);
    }
    sh.abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&sh.tmem, K::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  KvJobs<KvTile32Shared> jobs{sh.ring, &sh};
  bool lost = false;  // a result of this thread's is not finite

  if (warp == 0) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_f16(128, 128);
      constexpr uint32_t idesc_o = idesc_f16(128, D) | (1u << 16);  // B (V) MN-major
      bool ok = true;
      uint32_t n = 0, items = 0;
      for (;;) {
        KvJob it;
        ok = jobs.template take<false>(it, abort_flag);
        const int tiles = it.t1 - it.t0;
        if (!ok || tiles == 0) break;
        ok = mbar_wait(&sh.q_full, items & 1, abort_flag);
        for (int t = 0; ok && t < tiles; ++t, ++n) {
          const uint32_t ph = n & 1u;
          ok = mbar_wait(&sh.k_full, ph, abort_flag);
          if (!ok) break;
          tc_fence_after();
          // S' = Q' K'^T: hi.lo and lo.hi of all features, then hi.hi.  Every
          // addition to the accumulator is rounded at the size that the sum
          // has by then (towards zero): the small terms first leave a third
          // of the roundings at the full size.
          auto terms = [&](const uint8_t* q, const uint8_t* k, uint32_t first) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              if (kk * 16 >= c.d) break;
              const uint32_t off = (uint32_t)(kk >> 2) * K::PANEL + (uint32_t)(kk & 3) * 32;
              mma_f16(tmem + K::S_COL, desc_kmajor_sw128(smem_u32(q) + off), desc_kmajor_sw128(smem_u32(k) + off), idesc_s,
                      first && kk == 0 ? 0u : 1u);
            }
          };
          terms(q_hi, k_lo, 1u);
          terms(q_lo, k_hi, 0u);
          terms(q_hi, k_hi, 0u);
          tc_commit(&sh.s_full);
          tc_commit(&sh.k_empty);
          if (t + 1 == tiles) tc_commit(&sh.q_empty);
          // O' = P' V': wait for P, V, and for the previous O' to be read
          ok = mbar_wait(&sh.p_full, ph, abort_flag) && mbar_wait(&sh.v_full, ph, abort_flag) &&
               mbar_wait(&sh.o_empty, ph ^ 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          // P of keys [16 kk, 16 kk + 16): chunk kk / 2 of S's columns, hi in its first 16 columns, lo in the next 16
          auto products = [&](uint32_t lo, const uint8_t* v, uint32_t first) {
#pragma unroll
            for (int kk = 0; kk < K::BK / 16; ++kk)
              mma_f16_ta(tmem + K::O_COL, tmem + K::S_COL + lo + (uint32_t)(kk >> 1) * 32 + (uint32_t)(kk & 1) * 8,
                         desc_mnmajor_sw128(smem_u32(v) + (uint32_t)kk * 2048, K::PANEL, 1024), idesc_o, first && kk == 0 ? 0u : 1u);
          };
          products(0, v_lo, 1u);
          products(16, v_hi, 0u);
          products(0, v_hi, 0u);
          tc_commit(&sh.o_full);
          tc_commit(&sh.v_empty);
        }
        if (!ok) break;
        ++items;
        jobs.template drop<false>();
      }
      if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutMma);
    }
  } else if (warp <= kFaConv) {
    const int w = warp - 1, mine = w * 16 + (lane & 15);  // row whose offset this lane looks up
    const float ksign = a.scale2 < 0.0f ? -1.0f : 1.0f;
    const float* kb = static_cast<const float*>(c.k) + a.layer_off;
    const float* vb = static_cast<const float*>(c.v) + a.layer_off;
    bool ok = true;
    uint32_t n = 0, items = 0;
    for (;;) {
      KvJob it;
      ok = jobs.template take<true>(it, abort_flag);
      if (!ok || it.t0 == it.t1) break;
      ok = warp_wait(&sh.q_empty, (items & 1) ^ 1, abort_flag);
      if (!ok) break;
      const int rr = it.r0 + mine, token = plan_token(a.p, rr);
      const int64_t qoff = mine < it.rows ? (int64_t)(it.s.q0 + token) * a.qs + (int64_t)(it.h * a.p.group + rr - token * a.p.group) * c.d : -1;
      kv_convert_rows<D>(static_cast<const float*>(a.q), qoff, c.d, a.qvec, q_hi, q_lo, sh.icq[items & 1], 1.0f, w, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);
      int64_t next = kv_row_off(a, it.s.s, it.h, (it.tile0 + it.t0) * K::BK + mine, it.lo, it.hi);
      for (int t = it.t0; t < it.t1; ++t, ++n) {
        const uint32_t ph = n & 1u;
        const int64_t off = next;
        if (t + 1 < it.t1) next = kv_row_off(a, it.s.s, it.h, (it.tile0 + t + 1) * K::BK + mine, it.lo, it.hi);
        ok = warp_wait(&sh.k_empty, ph ^ 1u, abort_flag);
        if (!ok) break;
        kv_convert_rows<D>(kb, off, c.d, a.vec, k_hi, k_lo, sh.ick[ph], ksign, w, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.k_full);
        ok = warp_wait(&sh.v_empty, ph ^ 1u, abort_flag) &&
             kv_convert_values<D>(vb, off, c.d, a.vec, v_hi, v_lo, &sh.icv[ph], w, lane, sh.vpart[ph], &sh.vmax, ph, sh.short_of[ph],
                                  sh.uneven[ph], abort_flag);
        if (!ok) break;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.v_full);
      }
      if (!ok) break;
      ++items;
      jobs.template drop<true>();
    }
    if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutProducer);
  } else if (warp <= kFaConv + 4) {
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t unseen = a.scale2 < 0.0f ? 0x7f800000u : 0xff800000u;  // minus infinity once it has the key factors' sign
    bool ok = true;
    uint32_t n = 0, items = 0;
    for (;;) {
      KvJob it;
      ok = jobs.template take<true>(it, abort_flag);
      const int t0 = it.t0, t1 = it.t1;
      if (!ok || t0 == t1) break;
      int lo, hi;  // (rows behind the last see what it sees: masks are a whole warp's affair)
      plan_row_range(a.p, it.s, it.r0 + min(row, it.rows - 1), lo, hi);
      float rq2 = 0.0f;
      float m_i = -INFINITY, l_i = 0.0f;  // running max (log2 units) and 2^15-scaled sum
      for (int t = t0; t < t1; ++t, ++n) {
        const uint32_t ph = n & 1u;
        const int key0 = (it.tile0 + t) * K::BK, from = lo - key0, to = hi - key0;  // keys of this tile that are seen
        const bool all = __all_sync(0xffffffffu, from <= 0 && to >= K::BK);
        const float* ik = sh.ick[ph];
        ok = warp_wait(&sh.s_full, ph, abort_flag);
        if (!ok) break;
        tc_fence_after();
        // |scale| * log2(e) / c_q; the sign of scale rides on the key factors.
        // (S was computed from the queries, so their factors are there too; the
        // barrier of the queries may be phases ahead of this warp by now.)
        // (A scale of zero as the least that keeps minus infinity what it is.)
        if (t == t0) rq2 = fmaxf(__fmul_rn(fabsf(a.scale2), sh.icq[items & 1][row]), 1.2e-38f);
        // pass 1: the tile's max of S' * sign / c_k (rq2 > 0 keeps the order)
        float tmax = -INFINITY;
#pragma unroll 1
        for (int cb = 0; cb < 4; ++cb) {
          uint32_t r[32];
          tmem_ld32(lanes + K::S_COL + cb * 32, r);
          tmem_ld_wait();
          if (!all) kv_mask_chunk(r, from - cb * 32, to - cb * 32, unseen);
          tmax = fa_max_chunk<false>(r, ik + cb * 32, 32, tmax);
        }
        const float tm = tmax == -INFINITY ? -INFINITY : __fmul_rn(tmax, rq2);
        const float new_m = fmaxf(m_i, tm);
        const float corr = (m_i == -INFINITY) ? 0.0f : fa_ex2(__fsub_rn(m_i, new_m));
        // pass 2: p, the tile's sum, P terms into tensor memory.  (Past |m'| =
        // 2^20 the rounding of 15 - m' can reach an exponent of 16, which no
        // f16 holds: such a row is not finite and computed again.)
        const float nb = new_m == -INFINITY ? 0.0f : __fsub_rn(15.0f, new_m);
        // V's factors are there: whether its terms are enough for this row
        // (kv_convert_values; the weights once more, in tiles that ask for it)
        ok = warp_wait(&sh.v_full, ph, abort_flag);
        if (!ok) break;
        bool lossy = false;
        if (*reinterpret_cast<const volatile uint64_t*>(sh.uneven[ph])) {
          float lacks = 0.0f;
#pragma unroll 1
          for (int cb = 0; cb < 4; ++cb) {
            uint32_t r[32];
            tmem_ld32(lanes + K::S_COL + cb * 32, r);
            tmem_ld_wait();
            if (!all) kv_mask_chunk(r, from - cb * 32, to - cb * 32, unseen);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              lacks = fmaf(fa_ex2(__fmaf_rn(__fmul_rn(__uint_as_float(r[j]), ik[cb * 32 + j]), rq2, nb)), sh.short_of[ph][cb * 32 + j], lacks);
          }
          lossy = lacks > 0.0f;
        }
        float psum = 0.0f;
#pragma unroll 1
        for (int cb = 0; cb < 4; ++cb) {
          uint32_t r[32];
          tmem_ld32(lanes + K::S_COL + cb * 32, r);
          tmem_ld_wait();
          uint32_t ph16[16], pl16[16];
          if (!all) kv_mask_chunk(r, from - cb * 32, to - cb * 32, unseen);
          psum = __fadd_rn(psum, fa_p_chunk<false>(r, ik + cb * 32, rq2, nb, 32, ph16, pl16));
          // over S' chunk cb, which this thread has read
          tmem_st16(lanes + K::S_COL + cb * 32, ph16);
          tmem_st16(lanes + K::S_COL + cb * 32 + 16, pl16);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full);
        l_i = __fmaf_rn(l_i, corr, psum);
        m_i = new_m;
        if (lossy) l_i = NAN;  // and stays so: the row is computed again
        // O' of this tile -> o = o * corr + O' / c_v
        ok = warp_wait(&sh.o_full, ph, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float iv = sh.icv[ph];
#pragma unroll 1
        for (int cb = 0; cb < D / 32; ++cb) {
          uint32_t r[32], o[32];
          tmem_ld32(lanes + K::O_COL + cb * 32, r);
          if (t > t0) tmem_ld32(lanes + K::A_COL + cb * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int f = 0; f < 32; ++f)
            o[f] = __float_as_uint(
                __fmaf_rn(__uint_as_float(r[f]), iv, t > t0 ? __fmul_rn(__uint_as_float(o[f]), corr) : 0.0f));
          tmem_st32(lanes + K::A_COL + cb * 32, o);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.o_empty);
      }
      if (!ok) break;
      const bool whole = t0 == 0 && t1 == it.units;
      const int rr = it.r0 + row, token = plan_token(a.p, rr);
      const float inv = l_i == 0.0f ? 0.0f : __fdiv_rn(1.0f, l_i);
      float* dst = whole ? static_cast<float*>(a.out) + (int64_t)(it.s.q0 + token) * a.os + (int64_t)(it.h * a.p.group + rr - token * a.p.group) * c.d
                         : plan_slot(a, blockIdx.x, t0 == 0 ? 1 : 0, D) + plan_slot_o(K::ROWS) + (size_t)row * D;
      const bool vec = !whole || a.ovec16;
      if (!whole && row < it.rows) {
        float* slot = plan_slot(a, blockIdx.x, t0 == 0 ? 1 : 0, D);
        slot[row] = m_i, slot[K::ROWS + row] = l_i;
      }
#pragma unroll 1
      for (int cb = 0; cb < D / 32; ++cb) {
        uint32_t o[32];
        tmem_ld32(lanes + K::A_COL + cb * 32, o);
        tmem_ld_wait();
        if (row < it.rows) {
#pragma unroll
          for (int f = 0; f < 32; f += 4) {
            if (whole && cb * 32 + f >= c.d) break;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[e] = __uint_as_float(o[f + e]);
              if (whole) {
                // the quotient with one rounding more than the division's
                y[e] = __fmul_rn(y[e], inv);
                lost |= !isfinite(y[e]);
              }
            }
            if (vec) {
              *reinterpret_cast<float4*>(dst + cb * 32 + f) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (cb * 32 + f + e < c.d) dst[cb * 32 + f + e] = y[e];
            }
          }
        }
      }
      __syncwarp();
      tc_fence_before();  // the running output's columns belong to these warps alone
      ++items;
      jobs.template drop<true>();
    }
    if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutEpilogue);
  } else {
    int64_t left = min(chunk, total - chunk * blockIdx.x);
    bool ok = true;
    for (uint32_t items = 0;; ++items) {
      const uint32_t at = items % kJobs, ph = (items / kJobs) & 1;
      ok = warp_wait(&sh.job_empty[at], ph ^ 1, abort_flag);
      if (!ok) break;
      const int t0 = cur.at, t1 = kv_hand_out(a, cur, left, chunk, &sh.ring[at], &sh.job_full[at]);
      if (t0 == t1) break;
      left -= t1 - t0;
      if (left > 0) plan_next(a.p, c, a.bt, cur);
    }
    if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutProducer);
  }
  tc_fence_before();
  if (__syncthreads_or(lost) && threadIdx.x == 0) plan_lost(a);
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, K::TMEM_COLS);
  }
  pdl_wait();
}

}  // namespace oc
