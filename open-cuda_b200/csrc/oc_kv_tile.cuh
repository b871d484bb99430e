// oc_kv_tile.cuh -- attention over the paged cache for chunks of new tokens,
// f16 and bf16, on the tcgen05 tensor cores.  D: head_dim, or 64 or 128 above
// it with zeros behind (TMA fills them in; they cost the product with V, not
// the scores).
//
// An item is 256 query rows (two sub-tiles of 128) of one kv head; it walks
// tiles of 128 keys.  Per tile and sub-tile:
//   S = Q K^T      128 x 128, K = d      (both operands in shared memory)
//   P = 2^(scale2 * S - m)               (softmax warps, TMEM -> TMEM)
//   O += P V       128 x d, K = 128 keys (P in tensor memory over S's
//                  columns, V in shared memory, read as rows of keys)
// Bound: a tile's products take 2200 cycles of the tensor pipe at d = 128 (69
// an instruction measured, 32 of them) and its 2 * 16384 exponentials 2048 of
// the transcendental units, so neither may wait for the other: while one
// sub-tile's softmax runs, the tensor cores do the other's products, and the
// product with V begins on three quarters of the weights.  What is left is
// the chain of a sub-tile (scores out of tensor memory 420 cycles, maximum
// 370, exponentials 1500, then its two products): 3900 cycles a tile by a
// clock record.  Measured: chunks of 1.9 to 2 k tokens over 14 to 16 k keys,
// 32 heads of 128 over 8, 1020 us a call = 0.89 PFLOP/s.  Not kept, all slower
// there: two threads a row (16 softmax warps, 96 registers: 1120 us),
// exponentials in part as polynomials on the multiply-add pipe (1060 to 1200),
// items of 128 rows whose tiles two softmax groups take in turn (1215: twice
// the keys' traffic).  O stays in tensor memory and is rescaled only when a row's
// maximum has grown by more than 2^8 since the last time (f16: 2^4; larger
// weights lose nothing): after the first tiles that is rare, so the softmax
// almost never waits for the accumulator.  (That, and the early start of the
// product, are published ideas of attention on this generation of GPUs.)
//
// 384 threads, one CTA an SM:
//   warp 0       TMEM allocator, MMA issuer (lane 0)
//   warps 1, 2   loaders of K and of V into 128-byte-swizzled tiles, two
//                stages each: a tile whose keys the sequence holds is a few
//                TMA boxes (a page and 64 features each, one a lane); its last
//                tile, and pages of fewer than 8 tokens, are rows by cp.async,
//                zeros in place of keys that are not there
//   warp 3       walks the CTA's run and hands its pieces to the others;
//                loader of the queries (TMA where 128 rows are whole tokens)
//   warps 4..7   softmax and output of rows 0..127: thread = row = TMEM lane
//   warps 8..11  the same of rows 128..255
// Tensor memory: S / P of the two sub-tiles [0, 128) and [128, 256), O
// [256, 256 + d) and [256 + d, 256 + 2d).  Every wait is bounded (oc_ptx.cuh).
//
// P is rounded once to the operands' type (bf16: 2^-9 at most, as much as the
// result's own rounding); sums and maxima are f32, the sum of P is taken
// before the rounding.  Rows that are not finite, or would not be once rounded,
// are computed again from the definition (kv_row_exact), by the merge kernel:
// here the other warps' waits would run out.  A zero weight does not hide a
// NaN or an infinity of a key that the row does not see.
#pragma once
#include "oc_flash_tc.cuh"
#include "oc_kv_mma.cuh"

namespace oc {

template <typename T_, int D_>
struct KvTile {
  using T = T_;
  static constexpr int D = D_, DP = D_, ROWS = 256, BK = 128, THREADS = 384;
  static constexpr int PANEL = 128 * 128;        // bytes of 64 features of 128 rows
  static constexpr int TILE = 128 * D * 2;       // bytes of 128 rows
  static constexpr int S_COL = 0, O_COL = 256, TMEM_COLS = 512;
  static constexpr size_t SMEM = 1024 + 6 * (size_t)TILE;  // Q (2), K (2), V (2)
  // O is rescaled when a row's maximum has grown by more than 2^GROW since the
  // last time, and weights carry a factor of 2^UNIT.  f16 ends at 2^16 and
  // steps by 2^-24 below 2^-14: the factor puts the steps at 2^-35 of the
  // row's largest weight (at 2^-24 the lost halves of 2^17 keys made 2^-8).
  // Measured, f16, 2 chunks over 15 to 16 k keys, 32 heads of 128 over 8:
  // growth of 2^4 1051 us, 2^2 (steps at 2^-37) 1078, 2^1 1115.
  static constexpr bool HALF = std::is_same<T, __half>::value;
  static constexpr float GROW = HALF ? 4.0f : 8.0f, UNIT = HALF ? 11.0f : 0.0f;
  // bf16 operands are format 1, f16 format 0 (instruction descriptor bits 7.. and 10..)
  static constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
};

// A piece of an item: its tiles [t0, t1) of `units`.  One warp walks the
// CTA's run and hands the pieces to the others, a few ahead.
struct KvJob {
  KvSeq s;
  int b, h, r0, rows, lo, hi, tile0, units, t0, t1;  // t0 == t1: the run is over
};
constexpr int kJobs = 4;

struct KvTileBars {
  uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_part[2], p_full[2], o_done[2], o_free[2];
  uint64_t job_full[kJobs], job_empty[kJobs];
};

// mbar_wait of a whole warp: all lanes go on, or all give up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ float kv_max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// A consumer's place in the ring of jobs; B has the barriers.
template <typename B>
struct KvJobs {
  const KvJob* ring;
  B* bar;
  uint32_t at = 0, phase = 0;
  // The next job; false when a wait gave up.  Whole warps, or one thread.
  template <bool WARP>
  __device__ __forceinline__ bool take(KvJob& j, volatile int* abort_flag) {
    const bool ok = WARP ? warp_wait(&bar->job_full[at], phase, abort_flag) : mbar_wait(&bar->job_full[at], phase, abort_flag);
    if (ok) j = ring[at];
    return ok;
  }
  // Done with it.
  template <bool WARP>
  __device__ __forceinline__ void drop() {
    if (WARP) __syncwarp();
    if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(&bar->job_empty[at]);
    if (++at == kJobs) at = 0, phase ^= 1;
  }
};

// The walking warp: hands out the piece at `cur` (none when nothing is left)
// and notes the cut behind the run.  Returns where the piece ends.
__device__ __forceinline__ int kv_hand_out(const KvAttn& a, const KvCursor& cur, int64_t left, int64_t chunk, KvJob* slot,
                                           uint64_t* full) {
  const int t0 = cur.at, t1 = left > 0 ? (int)min((int64_t)cur.it.units, t0 + left) : t0;
  if ((threadIdx.x & 31) == 0) {
    *slot = KvJob{cur.s, cur.b, cur.h, cur.it.r0, cur.it.rows, cur.it.lo, cur.it.hi, cur.it.tile0, cur.it.units, t0, t1};
    if (t0 == 0 && t0 < t1 && t1 < cur.it.units) plan_cut(a, cur, cur.it.units - t1, chunk);
    mbar_arrive(full);
  }
  return t1;
}

// 16-byte chunks of a 128-row tile: D / 8 lanes take a row, so a warp copies
// RPI rows an instruction.
template <typename K>
struct KvTileRows {
  static constexpr int LPR = K::D / 8, RPI = 32 / LPR;
  static __device__ __forceinline__ uint32_t off(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * K::PANEL) + sw128_off(row, chunk & 7);
  }
};

// One warp: the K or the V tiles of a run.  `box`: keys a TMA box holds, 0
// for pages that are too small.
template <typename K>
__device__ __forceinline__ bool kv_tile_load(const KvAttn& a, KvJobs<KvTileBars> jobs, const CUtensorMap* map, const typename K::T* pool,
                                             uint8_t* tiles, uint64_t* full, uint64_t* empty, int box, volatile int* abort_flag) {
  using T = typename K::T;
  using R = KvTileRows<K>;
  const KvView& c = a.c;
  const int lane = threadIdx.x & 31, my_row = lane / R::LPR, ch = lane % R::LPR;
  uint32_t n = 0;
  for (;;) {
    KvJob it;
    if (!jobs.take<true>(it, abort_flag)) return false;
    const int t0 = it.t0, t1 = it.t1;
    if (t0 == t1) return true;
    const int* row = c.table + (size_t)max(it.s.s, 0) * c.max_pages;
    // boxes of a tile: one per `box` keys and 64 features; lane b has box b
    // (there are at most 32: 128 keys in boxes of 8, two halves)
    constexpr int PANELS = K::D / 64;
    const int boxes = box ? PANELS * (K::BK / box) : 0;
    const int my_key = box ? (lane / PANELS) * box : 0, my_panel = lane % PANELS;
    auto page_of = [&](int t) {  // of this lane's box; -1: the tile goes row by row
      const int key = (it.tile0 + t) * K::BK;
      if (!box || key + K::BK > it.s.len) return -1;
      if (lane >= boxes) return 0;
      const int page = row[(key + my_key) >> c.ps_shift];
      return page >= 0 && page < c.pages ? page : -1;
    };
    int page = page_of(t0);
    for (int t = t0; t < t1; ++t, ++n) {
      const uint32_t st = n & 1;
      uint8_t* dst = tiles + st * K::TILE;
      const int next = t + 1 < t1 ? page_of(t + 1) : -1;  // asked for before the wait
      const int key0 = (it.tile0 + t) * K::BK;
      if (!warp_wait(&empty[st], ((n >> 1) & 1) ^ 1, abort_flag)) return false;
      if (__all_sync(0xffffffffu, page >= 0)) {
        if (lane == 0) mbar_arrive_expect_tx(&full[st], K::TILE);
        __syncwarp();
        if (lane < boxes) {
          const int y = (int)(a.layer_off / c.d) + (int)((((int64_t)page * c.hk + it.h) << c.ps_shift) +
                                                          ((key0 + my_key) & ((1 << c.ps_shift) - 1)));
          tma_load_2d(dst + my_panel * K::PANEL + my_key * 128, map, my_panel * 64, y, &full[st]);
        }
      } else {
#pragma unroll 1
        for (int x = 0; x < 128; x += 32) {
          const int64_t off = kv_row_off(a, it.s.s, it.h, key0 + x + lane, it.lo, it.hi);
#pragma unroll 4
          for (int y = 0; y < 32; y += R::RPI) {
            const int64_t o = __shfl_sync(0xffffffffu, off, y + my_row);
            const bool there = o >= 0 && ch * 8 < c.d;
            cp_async16_zfill(dst + R::off(x + y + my_row, ch), pool + (there ? o + ch * 8 : 0), there);
          }
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
      page = next;
    }
    jobs.drop<true>();
  }
}

template <typename K>
__global__ void __launch_bounds__(K::THREADS, 1)
    kv_tile_kernel(const __grid_constant__ KvAttn a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                   const __grid_constant__ CUtensorMap mq, int box, int qbox) {
  using T = typename K::T;
  using R = KvTileRows<K>;
  constexpr int D = K::D;
  extern __shared__ uint8_t raw[];
  __shared__ KvPlanShared plan;
  __shared__ KvTileBars bar;
  __shared__ KvJob ring[kJobs];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sv = base;                  // V first: its descriptors' reach stays inside the allocation
  uint8_t* sk = base + 2 * K::TILE;
  uint8_t* sq = base + 4 * K::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Behind the warp-level kernel of the same call there is nothing to wait for:
  // that one lets this one start after its own wait, so all that came before
  // is there, and the two write different rows.  The wait then comes last, so
  // that this grid's end is the end of both.
  if (!a.beside) pdl_wait();
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
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], 1);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], 1);
      mbar_init(&bar.v_empty[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_part[i], 4);
      mbar_init(&bar.p_full[i], 4);
      mbar_init(&bar.o_done[i], 1);
      mbar_init(&bar.o_free[i], 4);
    }
    for (int i = 0; i < kJobs; ++i) {
      mbar_init(&bar.job_full[i], 1);
      mbar_init(&bar.job_empty[i], 3 + 8);  // MMA issuer, two loaders, eight softmax warps
    }
    abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, K::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  KvJobs<KvTileBars> jobs{ring, &bar};
  bool lost = false;  // a result of this thread's is not finite

  if (warp == 0) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_f16(128, 128) | K::FMT;
      constexpr uint32_t idesc_o = idesc_f16(128, D) | K::FMT | (1u << 16);  // V: features run first
      uint32_t n = 0, items = 0;       // tiles and items so far
      uint32_t p_ph[2] = {0, 0}, of_ph[2] = {1, 1};
      auto scores = [&](int sub, uint32_t tile) {
        const uint32_t q0 = smem_u32(sq) + sub * K::TILE, k0 = smem_u32(sk) + (tile & 1) * K::TILE;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          if (kk * 16 >= c.d) break;  // (zeros behind head_dim)
          const uint32_t off = (uint32_t)(kk >> 2) * K::PANEL + (uint32_t)(kk & 3) * 32;
          mma_f16(tmem + K::S_COL + sub * 128, desc_kmajor_sw128(q0 + off), desc_kmajor_sw128(k0 + off), idesc_s, kk != 0);
        }
        tc_commit(&bar.s_full[sub]);
      };
      bool ok = true;
      for (;;) {
        KvJob it;
        ok = jobs.take<false>(it, abort_flag);
        const int tiles = it.t1 - it.t0, subs = it.rows > 128 ? 2 : 1;
        if (!ok || tiles == 0) break;
        ok = mbar_wait(&bar.q_full, items & 1, abort_flag) && mbar_wait(&bar.k_full[n & 1], (n >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        for (int s = 0; s < subs; ++s) scores(s, n);
        tc_commit(&bar.k_empty[n & 1]);
        if (tiles == 1) tc_commit(&bar.q_empty);
        for (int t = 0; ok && t < tiles; ++t, ++n) {
          const bool more = t + 1 < tiles;
          for (int s = 0; ok && s < subs; ++s) {
            if (s == 0) ok = mbar_wait(&bar.v_full[n & 1], (n >> 1) & 1, abort_flag);
            // the first product of an item overwrites O: its last reader is done
            if (ok && t == 0) {
              ok = mbar_wait(&bar.o_free[s], of_ph[s], abort_flag);
              of_ph[s] ^= 1;
            }
            ok = ok && mbar_wait(&bar.p_part[s], p_ph[s], abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t v0 = smem_u32(sv) + (n & 1) * K::TILE;
            auto product = [&](int kk) {  // 16 keys
              mma_f16_ta(tmem + K::O_COL + s * D, tmem + K::S_COL + s * 128 + kk * 8,
                         desc_mnmajor_sw128(v0 + kk * 2048, K::PANEL, 1024), idesc_o, t != 0 || kk != 0);
            };
#pragma unroll
            for (int kk = 0; kk < 6; ++kk) product(kk);
            ok = mbar_wait(&bar.p_full[s], p_ph[s], abort_flag);
            p_ph[s] ^= 1;
            if (!ok) break;
            tc_fence_after();
            product(6);
            product(7);
            tc_commit(&bar.o_done[s]);
            if (s == subs - 1) tc_commit(&bar.v_empty[n & 1]);
            if (more) {
              if (s == 0) {
                ok = mbar_wait(&bar.k_full[(n + 1) & 1], ((n + 1) >> 1) & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
              }
              scores(s, n + 1);
              if (s == subs - 1) {
                tc_commit(&bar.k_empty[(n + 1) & 1]);
                if (t + 2 == tiles) tc_commit(&bar.q_empty);
              }
            }
          }
        }
        if (!ok) break;
        ++items;
        jobs.drop<false>();
      }
      if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutMma);
    }
  } else if (warp <= 2) {
    const bool is_k = warp == 1;
    if (box && lane == 0) prefetch_tmap(is_k ? &mk : &mv);
    const T* pool = static_cast<const T*>(is_k ? c.k : c.v) + a.layer_off;
    if (!kv_tile_load<K>(a, jobs, is_k ? &mk : &mv, pool, is_k ? sk : sv, is_k ? bar.k_full : bar.v_full,
                         is_k ? bar.k_empty : bar.v_empty, box, abort_flag))
      kernel_fail(a.dev_status, abort_flag, kDevTimeoutProducer);
  } else if (warp == 3) {
    // walks the run: hands out each piece, then brings its queries
    int64_t left = min(chunk, total - chunk * blockIdx.x);
    if (qbox && lane == 0) prefetch_tmap(&mq);
    bool ok = true;
    for (uint32_t items = 0; ok; ++items) {
      const uint32_t at = items % kJobs, ph = (items / kJobs) & 1;
      ok = warp_wait(&bar.job_empty[at], ph ^ 1, abort_flag);
      if (!ok) break;
      const int t0 = cur.at, t1 = kv_hand_out(a, cur, left, chunk, &ring[at], &bar.job_full[at]);
      if (t0 == t1) break;
      ok = warp_wait(&bar.q_empty, (items & 1) ^ 1, abort_flag);
      if (!ok) break;
      const int subs = cur.it.rows > 128 ? 2 : 1;
      if (qbox) {  // 128 rows are all heads of the group of 128 / G tokens (what lies behind the last row is not used)
        if (lane == 0) mbar_arrive_expect_tx(&bar.q_full, subs * K::TILE);
        __syncwarp();
        if (lane < subs * (D / 64)) {
          const int sub = lane / (D / 64), panel = lane % (D / 64);
          tma_load_3d(sq + sub * K::TILE + panel * K::PANEL, &mq, panel * 64, cur.h * a.p.group,
                      cur.s.q0 + plan_token(a.p, cur.it.r0) + sub * qbox, &bar.q_full);
        }
      } else {
        const int my_row = lane / R::LPR, ch = lane % R::LPR;
#pragma unroll 1
        for (int x = 0; x < subs * 128; x += 32) {
          const int r = x + lane, rr = cur.it.r0 + r, token = plan_token(a.p, rr);  // zeros behind the last row
          const int64_t off = r < cur.it.rows ? (int64_t)(cur.s.q0 + token) * a.qs + (int64_t)(cur.h * a.p.group + rr - token * a.p.group) * c.d : -1;
#pragma unroll 4
          for (int y = 0; y < 32; y += R::RPI) {
            const int64_t o = __shfl_sync(0xffffffffu, off, y + my_row);
            const bool there = o >= 0 && ch * 8 < c.d;
            cp_async16_zfill(sq + (x >> 7) * K::TILE + R::off((x & 127) + y + my_row, ch), static_cast<const T*>(a.q) + (there ? o + ch * 8 : 0),
                             there);
          }
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.q_full);
      }
      left -= t1 - t0;
      if (left > 0) plan_next(a.p, c, a.bt, cur);
    }
    if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutProducer);
  } else {
    const int sub = (warp - 4) >> 2, quad = warp & 3, row = sub * 128 + quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_col = tmem + K::S_COL + sub * 128 + lanes, o_col = tmem + K::O_COL + sub * D + lanes;
    const float sc = a.scale2 == 0.0f ? 1.0f : fabsf(a.scale2);
    uint32_t ph = 0, od = 0;  // phases of s_full and of o_done (one each a tile)
    bool ok = true;
    for (;;) {
      KvJob it;
      ok = jobs.take<true>(it, abort_flag);
      const int t0 = it.t0, t1 = it.t1;
      if (!ok || t0 == t1) break;
      const bool active = it.rows > sub * 128;  // the whole warp group
      if (active) {
        int lo = 0, hi = 0;
        if (row < it.rows) plan_row_range(a.p, it.s, it.r0 + row, lo, hi);
        // keys that all rows of the sub-tile see
        int all_lo, all_hi, unused;
        plan_row_range(a.p, it.s, it.r0 + sub * 128, unused, all_hi);
        plan_row_range(a.p, it.s, it.r0 + min(it.rows, sub * 128 + 128) - 1, all_lo, unused);
        float m = -INFINITY, l = 0.0f;  // log2 units
        for (int t = t0; t < t1; ++t) {
          const int key0 = (it.tile0 + t) * K::BK;
          ok = warp_wait(&bar.s_full[sub], ph, abort_flag);
          ph ^= 1;
          if (!ok) break;
          tc_fence_after();
          uint32_t s[128];
#pragma unroll
          for (int x = 0; x < 4; ++x) tmem_ld32(s_col + x * 32, *reinterpret_cast<uint32_t(*)[32]>(s + x * 32));
          tmem_ld_wait();
          if (a.scale2 <= 0.0f) {  // the sign goes to the scores; a scale of zero leaves zeros (and NaN of infinities)
            const float by = a.scale2 < 0.0f ? -1.0f : 0.0f;
#pragma unroll
            for (int x = 0; x < 128; ++x) s[x] = __float_as_uint(__uint_as_float(s[x]) * by);
          }
          if (key0 < all_lo || key0 + K::BK > all_hi) {
            const int from = lo - key0, to = hi - key0;  // of this row, within the tile
#pragma unroll
            for (int x = 0; x < 128; ++x)
              if (x < from || x >= to) s[x] = 0xff800000u;  // minus infinity
          }
          float mx[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) mx[x] = __uint_as_float(s[x]);
#pragma unroll
          for (int x = 4; x < 124; x += 8)
#pragma unroll
            for (int y = 0; y < 4; ++y) mx[y] = kv_max3(mx[y], __uint_as_float(s[x + 2 * y]), __uint_as_float(s[x + 2 * y + 1]));
#pragma unroll
          for (int y = 0; y < 4; ++y) mx[y] = fmaxf(mx[y], __uint_as_float(s[124 + y]));
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float mn = top == -INFINITY ? m : fmaxf(m, top * sc);
          if (__any_sync(0xffffffffu, mn > m + K::GROW)) {
            const float corr = mn == -INFINITY ? 1.0f : kv_ex2(m - mn);
            m = mn;
            l *= corr;
            if (t > t0) {
              // O holds the tiles so far: wait for the last product, scale it
              ok = warp_wait(&bar.o_done[sub], od ^ 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int x = 0; x < D; x += 16) {
                uint32_t o[16];
                tmem_ld16(o_col + x, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                tmem_st16(o_col + x, o);
              }
              tmem_st_wait();
            }
          }
          const float nb = m == -INFINITY ? 0.0f : K::UNIT - m;
          const uint64_t sc2 = f2_pack(sc, sc), nb2 = f2_pack(nb, nb);
          uint64_t sum2[2] = {0, 0};  // two pairs of f32 zeros
#pragma unroll
          for (int x0 = 0; x0 < 128; x0 += 32) {
            uint32_t p[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              float p0, p1;
              f2_unpack(f2_fma(u2_pack(s[x0 + x], s[x0 + x + 1]), sc2, nb2), p0, p1);
              p0 = kv_ex2(p0);
              p1 = kv_ex2(p1);
              sum2[(x >> 1) & 1] = f2_add(sum2[(x >> 1) & 1], f2_pack(p0, p1));
              p[x >> 1] = kv_pack2<T>(p0, p1);
            }
            tmem_st16(s_col + x0 / 2, p);
            if (x0 == 64) {  // three quarters of the product may begin
              tmem_st_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bar.p_part[sub]);
            }
          }
          {
            float x0, x1;
            f2_unpack(f2_add(sum2[0], sum2[1]), x0, x1);
            l += x0 + x1;
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.p_full[sub]);
          od ^= 1;
        }
        if (!ok) break;
        ok = warp_wait(&bar.o_done[sub], od ^ 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const bool whole = t0 == 0 && t1 == it.units;
        if (whole) {
          const int rr = it.r0 + row, token = plan_token(a.p, rr);
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          T* out = static_cast<T*>(a.out) + (int64_t)(it.s.q0 + token) * a.os +
                   (int64_t)(it.h * a.p.group + rr - token * a.p.group) * c.d;
#pragma unroll 1
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tmem_ld32(o_col + x, o);
            tmem_ld_wait();
            if (row < it.rows) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                if (x + e >= c.d) break;
                uint32_t p[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float y0 = __uint_as_float(o[e + 2 * k]) * inv, y1 = __uint_as_float(o[e + 2 * k + 1]) * inv;
                  lost |= kv_lost<T>(y0) || kv_lost<T>(y1);
                  p[k] = kv_pack2<T>(y0, y1);
                }
                if (a.ovec16) {
                  *reinterpret_cast<uint4*>(out + x + e) = make_uint4(p[0], p[1], p[2], p[3]);
                } else {
#pragma unroll
                  for (int k = 0; k < 8; ++k) out[x + e + k] = reinterpret_cast<const T*>(p)[k];
                }
              }
            }
          }
        } else {
          float* slot = plan_slot(a, blockIdx.x, t0 == 0 ? 1 : 0, D);
          if (row < it.rows) slot[row] = m, slot[K::ROWS + row] = l;
          float* po = slot + plan_slot_o(K::ROWS) + (size_t)row * D;
#pragma unroll 1
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tmem_ld32(o_col + x, o);
            tmem_ld_wait();
            if (row < it.rows)
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<uint4*>(po + x + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.o_free[sub]);
      }
      jobs.drop<true>();
    }
    if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutEpilogue);
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
