// oc_kv_append.cu -- oc_kv_append: the norms of queries and keys per head and
// the rotation by position in one pass over a token's projections, the keys
// and values written straight to their cache pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t),
//   t = position * inv_freq[j]
//
// Nothing is computed that memory would wait for, so the bound is the bytes:
// each element is read once and written once, 16 bytes a lane.  Few tokens: a
// CTA for a share of a token's heads (latency: 2.8 us for one token of 36
// heads of 128, a chain of four trips to memory); many: a warp a token (7967
// tokens, 147 MB, 40 us = 4.0 TB/s; about 100 instructions a row of a head
// keep it from the copy rate: 254 of them took 62 us).  The cosines and sines
// are computed once a token, in turns: t / (2 pi) in f64, reduced to
// [-1/2, 1/2] exactly before sincospif, so an angle of a far position keeps
// f32 accuracy (f32 products lose 1e-2 at position 1e5).  A
// lane holds eight features of a head that contain both members of its pairs
// (j and j + rot_dim / 2 as two runs of four), so the rotation needs no
// exchange, and a group of lanes that holds one head sums the squares with
// shuffles.  f32 throughout, one rounding when a result is stored.
#include "oc_kv.cuh"

namespace oc {

struct KvAppend {
  KvView c;
  KvBatch bt;
  size_t layer_off;  // elements before the layer in each pool
  const void *q, *k, *v, *qw, *kw;
  void* qo;
  int64_t qs, ks, vs, os;
  const float* inv_freq;
  float eps;
  int hq, rot, rows_per_cta;
};

constexpr int kAppendThreads = 256;

// The eight features of lane `u` of a head's group.  Pairs are (a[i], b[i]).
// Half-split rotation: a = features 4u .. 4u + 3, b = the same + rot / 2;
// past the rotated ones, and for interleaved pairs, eight consecutive ones.
template <typename T, bool SPLIT>
struct Octet {
  using Quad = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;  // four features
  struct Raw {
    Quad lo, hi;
  };
  static __device__ __forceinline__ void load(const T* x, int u, int rot, Raw& r) {
    const bool pairs = SPLIT && 8 * u < rot;
    r.lo = *reinterpret_cast<const Quad*>(x + (pairs ? 4 * u : 8 * u));
    r.hi = *reinterpret_cast<const Quad*>(x + (pairs ? rot / 2 + 4 * u : 8 * u + 4));
  }
  static __device__ __forceinline__ void values(const Raw& r, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
      const float* p = reinterpret_cast<const float*>(&r);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = p[i];
    } else {
      const uint32_t p[4] = {r.lo.x, r.lo.y, r.hi.x, r.hi.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = kv_unpack2<T>(p[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  }
  static __device__ __forceinline__ void norm(float (&f)[8], float inv, const Raw& weight) {
    float w[8];
    values(weight, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * w[e];
  }
  // Pair e of the four, by cosine and sine.
  static __device__ __forceinline__ void turn(float (&f)[8], int e, float2 g) {
    const int p = SPLIT ? e : 2 * e, q = SPLIT ? e + 4 : 2 * e + 1;
    const float x = f[p], y = f[q];
    f[p] = x * g.x - y * g.y;
    f[q] = y * g.x + x * g.y;
  }
  static __device__ __forceinline__ void store(T* y, int u, int rot, const Raw& r) {
    const bool pairs = SPLIT && 8 * u < rot;
    *reinterpret_cast<Quad*>(y + (pairs ? 4 * u : 8 * u)) = r.lo;
    *reinterpret_cast<Quad*>(y + (pairs ? rot / 2 + 4 * u : 8 * u + 4)) = r.hi;
  }
  static __device__ __forceinline__ void store(T* y, int u, int rot, const float (&f)[8]) {
    Raw r;
    if constexpr (sizeof(T) == 4) {
      r.lo = make_float4(f[0], f[1], f[2], f[3]);
      r.hi = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      r.lo = make_uint2(kv_pack2<T>(f[0], f[1]), kv_pack2<T>(f[2], f[3]));
      r.hi = make_uint2(kv_pack2<T>(f[4], f[5]), kv_pack2<T>(f[6], f[7]));
    }
    store(y, u, rot, r);
  }
};

// The sum of squares of a head, from its lanes' eight features each.
template <int LPR>
__device__ __forceinline__ float group_sum(const float (&f)[8]) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return ss;
}

// Where the token of a CTA belongs.
struct KvToken {
  int entry;      // of the batch, -1: behind the last sequence
  int seq, pos;   // row of the page table (-1: no such), position (negative: fewer tokens held than new)
  int64_t place;  // row of its kv head 0 in a layer's pool, -1: none
};

// cos and sin of pos * inv_freq[j].
__device__ __forceinline__ float2 kv_angle(int pos, float inv_freq) {
  const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;
  const float h = (float)(turns - rint(turns));  // in [-1/2, 1/2]
  float2 r;
  sincospif(2.0f * h, &r.y, &r.x);
  return r;
}

// All threads: finds token t, and in the same two block barriers fills cs with
// the cosines and sines of its rot / 2 angles.  An entry whose sequence stands
// earlier in the list as well is refused (two entries would write the same
// places).  False: nothing to do.
__device__ __forceinline__ bool kv_find_token(const KvAppend& a, int t, KvToken* sh, float2* cs) {
  const KvView& c = a.c;
  const KvBatch& bt = a.bt;
  // every thread looks at its entries at once; the one that has the token
  // goes on to its length (the entries are apart, so no two match unless cu
  // is not increasing: then any of them)
  if (threadIdx.x == 0) sh->entry = -1;
  __syncthreads();
  int my_seq = -1;  // of the last entry that this thread looked at
  for (int b = threadIdx.x; b < bt.n; b += blockDim.x) {
    const int q0 = bt.cu ? bt.cu[b] : b, q1 = bt.cu ? bt.cu[b + 1] : b + 1;
    my_seq = bt.seqs ? bt.seqs[b] : b;
    if (q0 <= t && t < q1) {
      const KvSeq s = kv_seq(c, bt, b);
      sh->seq = s.s;
      sh->pos = s.len - s.nq + (t - s.q0);
      sh->entry = b;
    }
  }
  __syncthreads();
  const int entry = sh->entry, seq = sh->seq, pos = sh->pos;
  if (entry < 0) return false;
  int twice = 0;
  if (bt.seqs) {
    if (bt.n <= (int)blockDim.x) {
      twice = (int)threadIdx.x < entry && my_seq == seq;
    } else {
      for (int b = threadIdx.x; b < entry; b += blockDim.x) twice |= bt.seqs[b] == seq;
    }
  }
  if (threadIdx.x < a.rot / 2) cs[threadIdx.x] = kv_angle(pos, a.inv_freq[threadIdx.x]);
  if (threadIdx.x == blockDim.x - 1) {
    int page = -1;
    if (seq >= 0 && pos >= 0) page = c.table[(size_t)seq * c.max_pages + (pos >> c.ps_shift)];
    const bool there = page >= 0 && page < c.pages;
    sh->place = there ? ((int64_t)page * c.hk << c.ps_shift) + (pos & ((1 << c.ps_shift) - 1)) : -1;
    if (seq >= 0 && !there) atomicOr(c.status, kKvBadPage);
  }
  twice = __syncthreads_or(twice);
  if (seq < 0 || twice) {
    if (threadIdx.x == 0) atomicOr(c.status, kKvBadSeq);
    return false;
  }
  return true;
}

// blockIdx.x = token, blockIdx.y = share of its rows (heads of q, k and v).
// LPR lanes per row, head_dim and rot_dim multiples of 8, rows of the inputs
// and pools aligned to 4 elements.  For few tokens: each thread has one octet,
// requested first, so that it is on its way while the token's place is looked up.
template <typename T, int LPR, bool SPLIT>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(KvAppend a) {
  __shared__ KvToken token;
  __shared__ float2 cs[128];
  using Oct = Octet<T, SPLIT>;
  pdl_wait();
  const KvView& c = a.c;
  const int t = blockIdx.x, d = c.d, rows = a.hq + 2 * c.hk, u = threadIdx.x % LPR;
  const int row0 = blockIdx.y * a.rows_per_cta, row1 = min(rows, row0 + a.rows_per_cta);
  const int r = row0 + threadIdx.x / LPR;  // rows_per_cta: one row a group of lanes
  const bool live = 8 * u < d && r < row1;
  const bool is_q = r < a.hq, is_k = !is_q && r < a.hq + c.hk;
  const int h = is_q ? r : is_k ? r - a.hq : r - a.hq - c.hk;
  const int rot = is_q || is_k ? a.rot : 0;
  const T* w = static_cast<const T*>(is_q ? a.qw : is_k ? a.kw : nullptr);
  typename Oct::Raw raw, rw;
  if (live) {
    const T* x = is_q   ? static_cast<const T*>(a.q) + (int64_t)t * a.qs
                 : is_k ? static_cast<const T*>(a.k) + (int64_t)t * a.ks
                        : static_cast<const T*>(a.v) + (int64_t)t * a.vs;
    Oct::load(x + (int64_t)h * d, u, rot, raw);
    if (w) Oct::load(w, u, rot, rw);
  }
  if (!kv_find_token(a, t, &token, cs)) return;
  const int64_t place = token.place;
  float f[8] = {};
  if (live) Oct::values(raw, f);
  const float ss = group_sum<LPR>(f);
  if (!live || (!is_q && place < 0)) return;
  if (w) Oct::norm(f, rsqrtf(ss / (float)d + a.eps), rw);
  if (8 * u < rot) {
#pragma unroll
    for (int e = 0; e < 4; ++e) Oct::turn(f, e, cs[4 * u + e]);
  }
  T* y = is_q ? static_cast<T*>(a.qo) + (int64_t)t * a.os + (int64_t)h * d
              : static_cast<T*>(is_k ? c.k : c.v) + a.layer_off + (size_t)(place + ((int64_t)h << c.ps_shift)) * d;
  Oct::store(y, u, rot, f);
}

// The same for many tokens: a warp a token, nothing shared, no barrier.  A
// lane's place within a head is the same for all heads, so it keeps the norms'
// weights and the cosines and sines of its four pairs in registers, and the
// rows of a token are one stream of loads with the lookup behind the first.
template <typename T, int LPR, bool SPLIT>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_warp_kernel(KvAppend a) {
  using Oct = Octet<T, SPLIT>;
  pdl_wait();
  const KvView& c = a.c;
  const int lane = threadIdx.x & 31, u = lane % LPR, d = c.d;
  const int t = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (t >= a.bt.total) return;
  constexpr int RPS = 32 / LPR, AT_ONCE = sizeof(T) == 4 ? 3 : 4;  // rows a step, steps a request
  typename Oct::Raw raw[AT_ONCE];
  const bool mine = 8 * u < d;
  const int first = lane / LPR;
  auto request = [&](const T* x, int r0, int n, int rot) {  // of n heads at x
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int r = r0 + i * RPS + first;
      if (mine && r < n) Oct::load(x + r * d, u, rot, raw[i]);
    }
  };
  const T* xq = static_cast<const T*>(a.q) + (int64_t)t * a.qs;
  request(xq, 0, a.hq, a.rot);
  // the last entry that begins at or before the token: 32 candidates a round
  const KvBatch& bt = a.bt;
  int entry = t;
  if (bt.cu) {
    entry = 0;
    for (int size = bt.n; size > 1;) {
      const int stride = (size + 31) / 32, b = entry + lane * stride;
      const uint32_t before = __ballot_sync(0xffffffffu, lane * stride < size && bt.cu[b] <= t);
      const int k = before ? 31 - __clz(before) : 0;
      size = min(stride, size - k * stride);
      entry += k * stride;
    }
    if (!(bt.cu[entry] <= t && t < bt.cu[entry + 1])) return;  // behind the last sequence
  } else if (t >= bt.n) {
    return;
  }
  const KvSeq s = kv_seq(c, bt, entry);
  const int pos = s.len - s.nq + (t - s.q0);
  bool twice = false;
  if (bt.seqs)
    for (int b = lane; b < entry; b += 32) twice |= bt.seqs[b] == s.s;
  int page = -1;
  if (s.s >= 0 && pos >= 0) page = c.table[(size_t)s.s * c.max_pages + (pos >> c.ps_shift)];
  if (__any_sync(0xffffffffu, twice) || s.s < 0) {
    if (lane == 0) atomicOr(c.status, kKvBadSeq);
    return;
  }
  const bool there = page >= 0 && page < c.pages;
  if (!there && lane == 0) atomicOr(c.status, kKvBadPage);
  const int64_t place = ((int64_t)page * c.hk << c.ps_shift) + (pos & ((1 << c.ps_shift) - 1));
  float2 cs[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (8 * u < a.rot) cs[e] = kv_angle(pos, a.inv_freq[4 * u + e]);
  const float per_d = 1.0f / (float)d;
  // n heads at x, norm and rotation, to y, `step` apart
  auto turn = [&](const T* x, T* y, int n, int64_t step, const T* weight, bool asked) {
    float w[8];
    if (weight && mine) {
      typename Oct::Raw rw;
      Oct::load(weight, u, a.rot, rw);
      Oct::values(rw, w);
    }
    for (int r0 = 0; r0 < n; r0 += AT_ONCE * RPS) {
      if (!asked || r0 > 0) request(x, r0, n, a.rot);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        if (r0 + i * RPS >= n) break;
        const int r = r0 + i * RPS + first;
        const bool live = mine && r < n;
        float f[8] = {};
        if (live) Oct::values(raw[i], f);
        if (weight) {
          const float inv = rsqrtf(fmaf(group_sum<LPR>(f), per_d, a.eps));
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * w[e];
        }
        if (8 * u < a.rot)
#pragma unroll
          for (int e = 0; e < 4; ++e) Oct::turn(f, e, cs[e]);
        if (live) Oct::store(y + r * step, u, a.rot, f);
      }
    }
  };
  turn(xq, static_cast<T*>(a.qo) + (int64_t)t * a.os, a.hq, d, static_cast<const T*>(a.qw), true);
  if (!there) return;
  const int64_t head = (int64_t)d << c.ps_shift;
  turn(static_cast<const T*>(a.k) + (int64_t)t * a.ks, static_cast<T*>(c.k) + a.layer_off + place * d, c.hk, head, static_cast<const T*>(a.kw), false);
  const T* xv = static_cast<const T*>(a.v) + (int64_t)t * a.vs;
  T* yv = static_cast<T*>(c.v) + a.layer_off + place * d;
  for (int r0 = 0; r0 < c.hk; r0 += AT_ONCE * RPS) {
    request(xv, r0, c.hk, 0);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int r = r0 + i * RPS + first;
      if (mine && r < c.hk) Oct::store(yv + r * head, u, 0, raw[i]);
    }
  }
}

// Any head_dim, rot_dim, stride and alignment: a warp per row, element loads.
// Lane l holds pairs l, l + 32, ... of the row: first the rotated pairs, then
// the remaining features two by two.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv_append_any_kernel(KvAppend a, int interleaved) {
  __shared__ KvToken token;
  __shared__ float2 cs[128];
  pdl_wait();
  const KvView& c = a.c;
  const int t = blockIdx.x, d = c.d;
  if (!kv_find_token(a, t, &token, cs)) return;
  const int64_t place = token.place;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.y * a.rows_per_cta, row1 = min(a.hq + 2 * c.hk, row0 + a.rows_per_cta);
  for (int r = row0 + warp; r < row1; r += kAppendThreads / 32) {
    const bool is_q = r < a.hq, is_k = !is_q && r < a.hq + c.hk;
    const int h = is_q ? r : is_k ? r - a.hq : r - a.hq - c.hk;
    const T* x = (is_q ? static_cast<const T*>(a.q) + (int64_t)t * a.qs
                       : is_k ? static_cast<const T*>(a.k) + (int64_t)t * a.ks : static_cast<const T*>(a.v) + (int64_t)t * a.vs) +
                 (int64_t)h * d;
    const int rot = is_q || is_k ? a.rot : 0, half = rot / 2;
    const T* w = static_cast<const T*>(is_q ? a.qw : is_k ? a.kw : nullptr);
    float f[4], g[4];
    int fi[4], gi[4];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = lane + 32 * i;
      if (p < half) {
        fi[i] = interleaved ? 2 * p : p;
        gi[i] = interleaved ? 2 * p + 1 : p + half;
      } else {
        fi[i] = rot + 2 * (p - half);
        gi[i] = fi[i] + 1;
      }
      f[i] = fi[i] < d ? kv_f32(x[fi[i]]) : 0.0f;
      g[i] = gi[i] < d ? kv_f32(x[gi[i]]) : 0.0f;
      ss = fmaf(f[i], f[i], fmaf(g[i], g[i], ss));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    T* y;
    if (is_q) {
      y = static_cast<T*>(a.qo) + (int64_t)t * a.os + (int64_t)h * d;
    } else {
      if (place < 0) continue;
      y = static_cast<T*>(is_k ? c.k : c.v) + a.layer_off + (size_t)(place + ((int64_t)h << c.ps_shift)) * d;
    }
    const float inv = w ? rsqrtf(ss / (float)d + a.eps) : 1.0f;
    __syncwarp();  // q_out may be q: the row has been read
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (w) {
        if (fi[i] < d) f[i] = f[i] * inv * kv_f32(w[fi[i]]);
        if (gi[i] < d) g[i] = g[i] * inv * kv_f32(w[gi[i]]);
      }
      const int p = lane + 32 * i;
      if (p < half) {
        const float2 e = cs[p];
        const float m = f[i], n = g[i];
        f[i] = m * e.x - n * e.y;
        g[i] = n * e.x + m * e.y;
      }
      if (fi[i] < d) y[fi[i]] = kv_from<T>(f[i]);
      if (gi[i] < d) y[gi[i]] = kv_from<T>(g[i]);
    }
  }
}

template <typename T>
static int launch_append(KvAppend a, int interleaved, cudaStream_t s) {
  const int rows = a.hq + 2 * a.c.hk, d = a.c.d;
  auto quad = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T))) == 0; };
  const bool vec = d % 8 == 0 && a.rot % 8 == 0 && quad(a.q) && quad(a.k) && quad(a.v) && quad(a.qo) && quad(a.c.k) &&
                   quad(a.c.v) && quad(a.qw) && quad(a.kw) && a.qs % 4 == 0 && a.ks % 4 == 0 && a.vs % 4 == 0 && a.os % 4 == 0;
  const int lpr = !vec ? 32 : d <= 64 ? 8 : d <= 128 ? 16 : 32;
  const int step = kAppendThreads / lpr, steps = (rows + step - 1) / step;
  // few tokens: a token's rows over several CTAs, a step of them each; many: a
  // warp a token.  Measured, 48 heads of 128 in f16, the first against the
  // second: one token 2.5 us : 8.4, 64 tokens 3.0 : 10.2, 512 5.7 : 10.6,
  // 1024 9.1 : 10.8, 1536 12.6 : 12.5, 4096 32 : 22 (three CTAs a token)
  const bool spread = (int64_t)a.bt.total * steps <= 20 * (int64_t)std::max(1, sm_count());
  a.rows_per_cta = spread ? step : rows;
  const dim3 block(kAppendThreads);
  auto go = [&](auto kern, dim3 grid) {
    OC_CHECK_CUDA(launch_pdl_ex(kern, grid, block, 0, s, a));
    return OC_OK;
  };
  if (!vec) {
    OC_CHECK_CUDA(launch_pdl_ex(kv_append_any_kernel<T>, dim3(a.bt.total, spread ? steps : 1), block, 0, s, a, interleaved));
    return OC_OK;
  }
  auto pick = [&](auto lanes, auto split) {
    constexpr int LPR = decltype(lanes)::value;
    constexpr bool SPLIT = decltype(split)::value;
    if (spread) return go(kv_append_kernel<T, LPR, SPLIT>, dim3(a.bt.total, steps));
    return go(kv_append_warp_kernel<T, LPR, SPLIT>, dim3((a.bt.total + kAppendThreads / 32 - 1) / (kAppendThreads / 32)));
  };
  auto by_style = [&](auto lanes) {
    return interleaved ? pick(lanes, std::false_type()) : pick(lanes, std::true_type());
  };
  if (lpr == 8) return by_style(std::integral_constant<int, 8>());
  if (lpr == 16) return by_style(std::integral_constant<int, 16>());
  return by_style(std::integral_constant<int, 32>());
}

}  // namespace oc

using namespace oc;

extern "C" int oc_kv_append(const oc_kv_cache* cache, int layer, int tokens, int n, const int32_t* cu,
                            const int32_t* seqs, int q_heads, const void* q, int64_t q_stride, const void* k,
                            int64_t k_stride, const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride,
                            const void* q_weight, const void* k_weight, float eps, const float* inv_freq, int rot_dim,
                            int interleaved, void* stream) {
  KvView c;
  if (int rc = kv_view(cache, &c)) return rc;
  OC_REQUIRE(layer >= 0 && layer < c.layers, "kv_append: no such layer");
  OC_REQUIRE(tokens >= 0 && n >= 0 && q_heads >= 0, "kv_append: negative size");
  OC_REQUIRE(cu || n == tokens, "kv_append: without cu each sequence has one token");
  OC_REQUIRE(rot_dim >= 0 && rot_dim <= c.d && rot_dim % 2 == 0, "kv_append: rot_dim must be even, 0..head_dim");
  OC_REQUIRE(rot_dim == 0 || inv_freq, "kv_append: rotation needs inv_freq");
  if (tokens == 0 || n == 0) return OC_OK;
  OC_REQUIRE(k && v && (q_heads == 0 || (q && q_out)), "kv_append: NULL pointer");
  OC_REQUIRE(n <= c.max_seqs, "kv_append: more entries than sequences");
  OC_REQUIRE(((int64_t)q_heads + 2 * (int64_t)c.hk) * c.d <= INT_MAX, "kv_append: too many heads");
  const int64_t kd = (int64_t)c.hk * c.d, qd = (int64_t)q_heads * c.d;
  OC_REQUIRE(k_stride >= kd && v_stride >= kd && (q_heads == 0 || (q_stride >= qd && q_out_stride >= qd)),
             "kv_append: a token stride is shorter than its heads");
  const int64_t es = (int64_t)kv_esize(cache->dtype);
  if (q_heads) {
    const bool in_place = q_out == q && (q_out_stride == q_stride || tokens == 1);
    OC_REQUIRE(in_place || !kv_overlap(q, q_stride * es, qd * es, q_out, q_out_stride * es, qd * es, tokens),
               "kv_append: q_out overlaps q and is not q itself");
    OC_REQUIRE(!kv_overlap(k, k_stride * es, kd * es, q_out, q_out_stride * es, qd * es, tokens) &&
                   !kv_overlap(v, v_stride * es, kd * es, q_out, q_out_stride * es, qd * es, tokens),
               "kv_append: q_out overlaps k or v");
  }
  KvAppend a;
  a.c = c;
  a.bt = KvBatch{cu, seqs, n, tokens};
  a.layer_off = (((size_t)layer * c.pages * c.hk) << c.ps_shift) * c.d;
  a.q = q, a.k = k, a.v = v, a.qw = q_weight, a.kw = k_weight, a.qo = q_out;
  a.qs = q_heads ? q_stride : 0, a.ks = k_stride, a.vs = v_stride, a.os = q_heads ? q_out_stride : 0;
  a.inv_freq = inv_freq;
  a.eps = eps;
  a.hq = q_heads, a.rot = rot_dim, a.rows_per_cta = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->dtype == OC_KV_F32) return launch_append<float>(a, interleaved, s);
  if (cache->dtype == OC_KV_F16) return launch_append<__half>(a, interleaved, s);
  return launch_append<__nv_bfloat16>(a, interleaved, s);
}
