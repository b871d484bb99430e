// oc_kv_tile.cuh -- attention over the paged cache for chunks of new tokens,
// f16 and bf16, head_dim 64 and 128, on the tcgen05 tensor cores.
//
// An item is 256 query rows (two sub-tiles of 128) of one kv head; it walks
// tiles of 128 keys.  Per tile and sub-tile:
//   S = Q K^T      128 x 128, K = d      (both operands in shared memory)
//   P = 2^(scale2 * S - m)               (softmax warps, TMEM -> TMEM)
//   O += P V       128 x d, K = 128 keys (P in tensor memory over S's
//                  columns, V in shared memory, read as rows of keys)
// Bound: a tile is 2 * 2 * 128 * 128 * d multiply-adds per sub-tile (2048
// cycles of the tensor pipe for both at d = 128) and 2 * 16384 exponentials
// (2048 cycles at 16 a clock), so neither may wait for the other: while one
// sub-tile's softmax runs, the tensor cores do the other's products.  O stays
// in tensor memory and is rescaled only when a row's maximum grows by more
// than 2^8 since the last time (weights up to 2^8 are exact powers away from
// the usual ones, and both types hold them): after the first tiles that is
// rare, so the softmax almost never waits for the accumulator.
//
// 384 threads, one CTA an SM:
//   warp 0       TMEM allocator, MMA issuer (lane 0)
//   warps 1..3   loaders: rows of pages -> 128-byte-swizzled tiles by
//                cp.async (a page of any size, even one token, is a list of
//                rows), two stages each of K and V
//   warps 4..7   softmax and output of rows 0..127: thread = row = TMEM lane
//   warps 8..11  the same of rows 128..255
// Tensor memory: S / P of the two sub-tiles [0, 128) and [128, 256), O
// [256, 256 + d) and [256 + d, 256 + 2d).  Every wait is bounded (oc_ptx.cuh).
//
// P is rounded once to the operands' type (bf16: 2^-9 at most, as much as the
// result's own rounding); sums and maxima are f32, the sum of P is taken
// before the rounding.  Rows that are not finite are computed again from the
// definition (kv_row_exact): a zero weight does not hide a NaN or an infinity
// of a key that the row does not see.
#pragma once
#include "oc_flash_tc.cuh"
#include "oc_kv_mma.cuh"

namespace oc {

template <typename T_, int D_>
struct KvTile {
  using T = T_;
  static constexpr int D = D_, DP = D_, ROWS = 256, BK = 128, THREADS = 384;
  static constexpr int LOADERS = 3;
  static constexpr int PANEL = 128 * 128;        // bytes of 64 features of 128 rows
  static constexpr int TILE = 128 * D * 2;       // bytes of 128 rows
  static constexpr int S_COL = 0, O_COL = 256, TMEM_COLS = 512;
  static constexpr size_t SMEM = 1024 + 6 * (size_t)TILE;  // Q (2), K (2), V (2)
  // bf16 operands are format 1, f16 format 0 (instruction descriptor bits 7.. and 10..)
  static constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
};

struct KvTileBars {
  uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_done[2], o_free[2];
};

// mbar_wait of a whole warp: all lanes go on, or all give up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// The pieces of a CTA's run, walked alike by every role.
struct KvWalk {
  KvCursor cur;
  int64_t left;
  __device__ __forceinline__ int first() const { return cur.at; }
  __device__ __forceinline__ int last() const { return (int)min((int64_t)cur.it.units, cur.at + left); }
  __device__ __forceinline__ void next(const KvAttn& a, int done) {
    left -= done;
    if (left > 0) plan_next(a.p, a.c, a.bt, cur);
  }
};

// Row `r` (lane's share) of a 128-row tile: 16-byte chunks.  D / 8 lanes take
// a row, so a warp takes RPI rows an instruction.
template <typename K>
struct KvTileRows {
  static constexpr int LPR = K::D / 8, RPI = 32 / LPR, STEPS = 128 / RPI;
  static constexpr int MINE = (STEPS + K::LOADERS - 1) / K::LOADERS;  // instructions of one loader warp
  static constexpr int HELD = (MINE * RPI + 31) / 32;                 // offsets a lane keeps
  static __device__ __forceinline__ uint32_t off(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * K::PANEL) + sw128_off(row, chunk & 7);
  }
};

template <typename K>
__global__ void __launch_bounds__(K::THREADS, 1) kv_tile_kernel(KvAttn a) {
  using T = typename K::T;
  using R = KvTileRows<K>;
  constexpr int D = K::D;
  extern __shared__ uint8_t raw[];
  __shared__ KvPlanShared plan;
  __shared__ KvTileBars bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sv = base;                  // V first: its descriptors' reach stays inside the allocation
  uint8_t* sk = base + 2 * K::TILE;
  uint8_t* sq = base + 4 * K::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  const KvView& c = a.c;
  KvWalk w;
  int64_t chunk;
  const int64_t total = plan_locate(a.p, c, a.bt, blockIdx.x, &plan, &chunk, w.cur);
  if (threadIdx.x == 0) plan_no_cut(a);
  if (total == 0) return;
  w.left = min(chunk, total - chunk * blockIdx.x);
  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, K::LOADERS);
    mbar_init(&bar.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], K::LOADERS);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], K::LOADERS);
      mbar_init(&bar.v_empty[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i], 4);
      mbar_init(&bar.o_done[i], 1);
      mbar_init(&bar.o_free[i], 4);
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
          const uint32_t off = (uint32_t)(kk >> 2) * K::PANEL + (uint32_t)(kk & 3) * 32;
          mma_f16(tmem + K::S_COL + sub * 128, desc_kmajor_sw128(q0 + off), desc_kmajor_sw128(k0 + off), idesc_s, kk != 0);
        }
        tc_commit(&bar.s_full[sub]);
      };
      bool ok = true;
      while (ok && w.left > 0) {
        const int tiles = w.last() - w.first(), subs = w.cur.it.rows > 128 ? 2 : 1;
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
            ok = ok && mbar_wait(&bar.p_full[s], p_ph[s], abort_flag);
            p_ph[s] ^= 1;
            if (!ok) break;
            tc_fence_after();
            const uint32_t v0 = smem_u32(sv) + (n & 1) * K::TILE;
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              mma_f16_ta(tmem + K::O_COL + s * D, tmem + K::S_COL + s * 128 + kk * 8,
                         desc_mnmajor_sw128(v0 + kk * 2048, K::PANEL, 1024), idesc_o, t != 0 || kk != 0);
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
        ++items;
        w.next(a, tiles);
      }
      if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutMma);
    }
  } else if (warp <= K::LOADERS) {
    const int lw = warp - 1;
    const T* kb = static_cast<const T*>(c.k) + a.layer_off;
    const T* vb = static_cast<const T*>(c.v) + a.layer_off;
    const int my_row = lane / R::LPR, ch = lane % R::LPR;
    uint32_t n = 0, items = 0;
    // copies in flight, oldest first: which barrier each group completes.  A
    // group is announced two groups later (or at the end), when it has landed.
    uint64_t *b0 = nullptr, *b1 = nullptr;
    auto announce = [&](uint64_t* b) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    // Before this warp waits for room, what it has copied is announced: the
    // consumers may need exactly that to make room.
    auto take = [&](uint64_t* b, uint32_t parity) {
      if (__all_sync(0xffffffffu, mbar_try_wait(smem_u32(b), parity))) return true;
      cp_async_wait<0>();
      if (b0) announce(b0);
      if (b1) announce(b1);
      b0 = b1 = nullptr;
      return warp_wait(b, parity, abort_flag);
    };
    auto push = [&](uint64_t* b) {
      cp_async_commit();
      if (b0) {
        cp_async_wait<2>();
        announce(b0);
      }
      b0 = b1;
      b1 = b;
    };
    bool ok = true;
    while (ok && w.left > 0) {
      const KvItem& it = w.cur.it;
      const int t0 = w.first(), t1 = w.last();
      // queries: rows of the item, zeros behind the last
      ok = take(&bar.q_empty, (items & 1) ^ 1);
      if (!ok) break;
      const int q_rows = it.rows > 128 ? 256 : 128;
      for (int r0 = lw * R::RPI; r0 < q_rows; r0 += K::LOADERS * R::RPI) {
        const int r = r0 + my_row, rr = it.r0 + r, token = plan_token(a.p, rr);
        const bool there = r < it.rows;
        const T* src = static_cast<const T*>(a.q);
        if (there) src += (int64_t)(w.cur.s.q0 + token) * a.qs + (int64_t)(w.cur.h * a.p.group + rr - token * a.p.group) * D + ch * 8;
        cp_async16_zfill(sq + (r >> 7) * K::TILE + R::off(r & 127, ch), src, there);
      }
      push(&bar.q_full);
      // offsets of this warp's rows of a tile: instruction i of the warp has
      // rows (lw + LOADERS i) * RPI + lane / LPR; lane j keeps that of number j
      int64_t off[R::HELD], nxt[R::HELD];
      auto offsets = [&](int t, int64_t (&o)[R::HELD]) {
#pragma unroll
        for (int x = 0; x < R::HELD; ++x) {
          const int j = x * 32 + lane, i = j / R::RPI;
          const int row = (lw + K::LOADERS * i) * R::RPI + j % R::RPI;
          o[x] = t < t1 && row < 128 ? kv_row_off(a, w.cur.s.s, w.cur.h, (it.tile0 + t) * K::BK + row, it.lo, it.hi) : -1;
        }
      };
      auto copy = [&](const T* pool, uint8_t* dst) {
#pragma unroll
        for (int i = 0; i < R::MINE; ++i) {
          const int step = lw + K::LOADERS * i;
          const int64_t o = __shfl_sync(0xffffffffu, off[i * R::RPI / 32], (i * R::RPI) % 32 + my_row);
          if (step < R::STEPS) cp_async16_zfill(dst + R::off(step * R::RPI + my_row, ch), pool + (o < 0 ? 0 : o) + ch * 8, o >= 0);
        }
      };
      offsets(t0, off);
      for (int t = t0; t < t1; ++t, ++n) {
        const uint32_t st = n & 1, ph = ((n >> 1) & 1) ^ 1;
        offsets(t + 1, nxt);
        ok = take(&bar.k_empty[st], ph);
        if (!ok) break;
        copy(kb, sk + st * K::TILE);
        push(&bar.k_full[st]);
        ok = take(&bar.v_empty[st], ph);
        if (!ok) break;
        copy(vb, sv + st * K::TILE);
        push(&bar.v_full[st]);
#pragma unroll
        for (int x = 0; x < R::HELD; ++x) off[x] = nxt[x];
      }
      ++items;
      w.next(a, t1 - t0);
    }
    cp_async_wait<0>();
    if (ok) {
      if (b0) announce(b0);
      if (b1) announce(b1);
    } else {
      kernel_fail(a.dev_status, abort_flag, kDevTimeoutProducer);
    }
  } else {
    const int sub = (warp - 4) >> 2, quad = warp & 3, row = sub * 128 + quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_col = tmem + K::S_COL + sub * 128 + lanes, o_col = tmem + K::O_COL + sub * D + lanes;
    const float sc = fabsf(a.scale2);
    const bool flip = a.scale2 < 0.0f;
    uint32_t ph = 0, od = 0;  // phases of s_full and of o_done (one each a tile)
    bool ok = true;
    while (ok && w.left > 0) {
      const KvItem& it = w.cur.it;
      const int t0 = w.first(), t1 = w.last();
      const bool active = it.rows > sub * 128;  // the whole warp group
      if (active) {
        int lo = 0, hi = 0;
        if (row < it.rows) plan_row_range(a.p, w.cur.s, it.r0 + row, lo, hi);
        // keys that all rows of the sub-tile see
        int all_lo, all_hi, unused;
        plan_row_range(a.p, w.cur.s, it.r0 + sub * 128, unused, all_hi);
        plan_row_range(a.p, w.cur.s, it.r0 + min(it.rows, sub * 128 + 128) - 1, all_lo, unused);
        float m = -INFINITY, l = 0.0f;  // log2 units
        for (int t = t0; t < t1; ++t) {
          const int key0 = (it.tile0 + t) * K::BK;
          const bool masked = key0 < all_lo || key0 + K::BK > all_hi;
          const int from = lo - key0, to = hi - key0;  // of this row, within the tile
          ok = warp_wait(&bar.s_full[sub], ph, abort_flag);
          ph ^= 1;
          if (!ok) break;
          tc_fence_after();
          uint32_t s[128];
#pragma unroll
          for (int x = 0; x < 4; ++x) tmem_ld32(s_col + x * 32, *reinterpret_cast<uint32_t(*)[32]>(s + x * 32));
          tmem_ld_wait();
          if (flip)
#pragma unroll
            for (int x = 0; x < 128; ++x) s[x] ^= 0x80000000u;
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (masked) {
#pragma unroll
            for (int x = 0; x < 128; ++x)
              if (x >= from && x < to) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(s[x]));
          } else {
#pragma unroll
            for (int x = 0; x < 128; ++x) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(s[x]));
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float mn = top == -INFINITY ? m : fmaxf(m, top * sc);
          if (__any_sync(0xffffffffu, mn > m + 8.0f)) {
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
          const float nb = m == -INFINITY ? 0.0f : -m;
          float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          auto weigh = [&](int x) {
            const float p = kv_ex2(fmaf(__uint_as_float(s[x]), sc, nb));
            return p;
          };
#pragma unroll
          for (int x0 = 0; x0 < 128; x0 += 32) {
            uint32_t p[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              float p0 = weigh(x0 + x), p1 = weigh(x0 + x + 1);
              if (masked) {
                p0 = x0 + x >= from && x0 + x < to ? p0 : 0.0f;
                p1 = x0 + x + 1 >= from && x0 + x + 1 < to ? p1 : 0.0f;
              }
              sum[x & 2] += p0;
              sum[(x & 2) + 1] += p1;
              p[x >> 1] = kv_pack2<T>(p0, p1);
            }
            tmem_st16(s_col + x0 / 2, p);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
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
          T* out = static_cast<T*>(a.out) + (int64_t)(w.cur.s.q0 + token) * a.os +
                   (int64_t)(w.cur.h * a.p.group + rr - token * a.p.group) * D;
          bool bad = false;
#pragma unroll 1
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tmem_ld32(o_col + x, o);
            tmem_ld_wait();
            if (row < it.rows) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint32_t p[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float y0 = __uint_as_float(o[e + 2 * k]) * inv, y1 = __uint_as_float(o[e + 2 * k + 1]) * inv;
                  bad |= !isfinite(y0) || !isfinite(y1);
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
          __syncwarp();
          for (uint32_t todo = __ballot_sync(0xffffffffu, bad); todo; todo &= todo - 1)
            kv_row_exact<T>(a, w.cur.s, w.cur.h, it.r0 + sub * 128 + quad * 32 + __ffs(todo) - 1);
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
      if (threadIdx.x == 128 && t0 == 0 && t1 < it.units) plan_cut(a, w.cur, it.units - t1, chunk);
      w.next(a, t1 - t0);
    }
    if (!ok) kernel_fail(a.dev_status, abort_flag, kDevTimeoutEpilogue);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, K::TMEM_COLS);
  }
}

}  // namespace oc
