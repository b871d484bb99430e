// oc_kv_append.cu -- oc_kv_append: the norms of queries and keys per head and
// the rotation by position in one pass over a token's projections, the keys
// and values written straight to their cache pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t),
//   t = position * inv_freq[j]
//
// Nothing is computed twice that memory would wait for, so the bound is the
// bytes: each element is read once and written once, 16 bytes a lane.  One
// CTA works on one token (or, when there are few tokens, on a share of its
// heads); its cosines and sines are computed once, in turns: t / (2 pi) in
// f64, reduced to [-1/2, 1/2] exactly before sincospif, so an angle of a far
// position keeps f32 accuracy (f32 products lose 1e-2 at position 1e5).  A
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
  static __device__ __forceinline__ bool paired(int u, int rot) { return !SPLIT || 8 * u < rot; }
  static __device__ __forceinline__ void load(const T* x, int u, int rot, float (&f)[8]) {
    if (SPLIT && 8 * u < rot) {
      quad(x + 4 * u, f);
      quad(x + rot / 2 + 4 * u, f + 4);
    } else {
      quad(x + 8 * u, f);
      quad(x + 8 * u + 4, f + 4);
    }
  }
  static __device__ __forceinline__ void store(T* y, int u, int rot, const float (&f)[8]) {
    if (SPLIT && 8 * u < rot) {
      put(y + 4 * u, f);
      put(y + rot / 2 + 4 * u, f + 4);
    } else {
      put(y + 8 * u, f);
      put(y + 8 * u + 4, f + 4);
    }
  }
  static __device__ __forceinline__ void quad(const T* x, float* f) {
    if constexpr (sizeof(T) == 4) {
      const float4 r = *reinterpret_cast<const float4*>(x);
      f[0] = r.x, f[1] = r.y, f[2] = r.z, f[3] = r.w;
    } else {
      const uint2 r = *reinterpret_cast<const uint2*>(x);
      const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = kv_f32(p[i]);
    }
  }
  static __device__ __forceinline__ void put(T* y, const float* f) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(y) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      uint2 r;
      T* p = reinterpret_cast<T*>(&r);
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = kv_from<T>(f[i]);
      *reinterpret_cast<uint2*>(y) = r;
    }
  }
};

// Where the token of this CTA belongs; filled by kv_find_token.
struct KvToken {
  int pos;   // position in the sequence, negative when it holds fewer tokens than are new
  int seq;   // row of the page table
  bool ok;
};

// All threads: the entry whose new tokens contain token t.  An entry whose
// sequence stands earlier in the list as well is refused (two entries would
// write the same places).
__device__ __forceinline__ KvToken kv_find_token(const KvView& c, const KvBatch& bt, int t, int* slot) {
  KvToken r{0, -1, false};
  if (threadIdx.x == 0) *slot = -1;
  __syncthreads();
  if (bt.cu) {
    for (int b = threadIdx.x; b < bt.n; b += blockDim.x)
      if (bt.cu[b] <= t && t < bt.cu[b + 1]) atomicMax(slot, b);
  } else if (threadIdx.x == 0 && t < bt.n) {
    *slot = t;
  }
  __syncthreads();
  const int b = *slot;
  if (b < 0) return r;
  const KvSeq s = kv_seq(c, bt, b);
  int twice = 0;
  if (bt.seqs)
    for (int i = threadIdx.x; i < b; i += blockDim.x) twice |= bt.seqs[i] == s.s;
  twice = __syncthreads_or(twice);
  if (s.s < 0 || twice) {
    if (threadIdx.x == 0) atomicOr(c.status, kKvBadSeq);
    return r;
  }
  r.seq = s.s;
  r.pos = s.len - s.nq + (t - s.q0);
  r.ok = true;
  return r;
}

// cos and sin of pos * inv_freq[j].
__device__ __forceinline__ float2 kv_angle(int pos, float inv_freq) {
  const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;
  const float h = (float)(turns - rint(turns));  // in [-1/2, 1/2]
  float2 r;
  sincospif(2.0f * h, &r.y, &r.x);
  return r;
}

// Place of kv head 0 of the token in a layer's pool, or -1 without one.
__device__ __forceinline__ int64_t kv_place(const KvView& c, const KvToken& tk) {
  if (tk.pos < 0) {
    if (threadIdx.x == 0) atomicOr(c.status, kKvBadPage);
    return -1;
  }
  const int page = c.table[(size_t)tk.seq * c.max_pages + (tk.pos >> c.ps_shift)];
  if (page < 0 || page >= c.pages) {
    if (threadIdx.x == 0) atomicOr(c.status, kKvBadPage);
    return -1;
  }
  return ((int64_t)page * c.hk << c.ps_shift) + (tk.pos & ((1 << c.ps_shift) - 1));  // in rows of head_dim
}

// blockIdx.x = token, blockIdx.y = share of its rows (heads of q, k and v).
// LPR lanes per row, head_dim and rot_dim multiples of 8, rows of the inputs
// and pools aligned to 4 elements.
template <typename T, int LPR, bool SPLIT>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(KvAppend a) {
  __shared__ int slot;
  __shared__ float2 cs[128];
  pdl_wait();
  const KvView& c = a.c;
  const int t = blockIdx.x, d = c.d;
  const KvToken tk = kv_find_token(c, a.bt, t, &slot);
  if (!tk.ok) return;
  if (threadIdx.x < a.rot / 2) cs[threadIdx.x] = kv_angle(tk.pos, a.inv_freq[threadIdx.x]);
  const int64_t place = kv_place(c, tk);
  __syncthreads();
  const int rows = a.hq + 2 * c.hk, u = threadIdx.x % LPR;
  const int row0 = blockIdx.y * a.rows_per_cta, row1 = min(rows, row0 + a.rows_per_cta);
  const bool mine = 8 * u < d;
  constexpr int STEP = kAppendThreads / LPR;
  // whole warps iterate, so that the shuffles below have all their lanes
  for (int r0 = row0; r0 < row1; r0 += STEP) {
    const int r = r0 + threadIdx.x / LPR;
    const bool live = mine && r < row1;
    const bool is_q = r < a.hq, is_k = !is_q && r < a.hq + c.hk;
    const int h = is_q ? r : is_k ? r - a.hq : r - a.hq - c.hk;
    const T* x = is_q ? static_cast<const T*>(a.q) + (int64_t)t * a.qs
                      : is_k ? static_cast<const T*>(a.k) + (int64_t)t * a.ks : static_cast<const T*>(a.v) + (int64_t)t * a.vs;
    const int rot = is_q || is_k ? a.rot : 0;
    float f[8] = {};
    if (live) Octet<T, SPLIT>::load(x + (int64_t)h * d, u, rot, f);
    const T* w = static_cast<const T*>(is_q ? a.qw : is_k ? a.kw : nullptr);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!live) continue;
    if (w) {
      const float inv = rsqrtf(ss / (float)d + a.eps);
      float wf[8];
      Octet<T, SPLIT>::load(w, u, rot, wf);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * wf[i];
    }
    if (8 * u < rot) {
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = cs[4 * u + i];
          const float p = f[i], q = f[i + 4];
          f[i] = p * e.x - q * e.y;
          f[i + 4] = q * e.x + p * e.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = cs[4 * u + i];
          const float p = f[2 * i], q = f[2 * i + 1];
          f[2 * i] = p * e.x - q * e.y;
          f[2 * i + 1] = q * e.x + p * e.y;
        }
      }
    }
    T* y;
    if (is_q) {
      y = static_cast<T*>(a.qo) + (int64_t)t * a.os + (int64_t)h * d;
    } else {
      if (place < 0) continue;
      y = static_cast<T*>(is_k ? c.k : c.v) + a.layer_off + (size_t)(place + ((int64_t)h << c.ps_shift)) * d;
    }
    Octet<T, SPLIT>::store(y, u, rot, f);
  }
}

// Any head_dim, rot_dim, stride and alignment: a warp per row, element loads.
// Lane l holds pairs l, l + 32, ... of the row: first the rotated pairs, then
// the remaining features two by two.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv_append_any_kernel(KvAppend a, int interleaved) {
  __shared__ int slot;
  __shared__ float2 cs[128];
  pdl_wait();
  const KvView& c = a.c;
  const int t = blockIdx.x, d = c.d;
  const KvToken tk = kv_find_token(c, a.bt, t, &slot);
  if (!tk.ok) return;
  if (threadIdx.x < a.rot / 2) cs[threadIdx.x] = kv_angle(tk.pos, a.inv_freq[threadIdx.x]);
  const int64_t place = kv_place(c, tk);
  __syncthreads();
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
  // few tokens: a token's rows over several CTAs, each with one step of them
  // (one token of 36 heads: 3 CTAs); many: one CTA, its angles computed once
  const bool spread = (int64_t)a.bt.total * steps <= 4 * (int64_t)std::max(1, sm_count());
  const int shares = spread ? steps : 1;
  a.rows_per_cta = spread ? step : rows;
  const dim3 grid(a.bt.total, shares), block(kAppendThreads);
  auto go = [&](auto kern) {
    OC_CHECK_CUDA(launch_pdl_ex(kern, grid, block, 0, s, a));
    return OC_OK;
  };
  if (!vec) {
    OC_CHECK_CUDA(launch_pdl_ex(kv_append_any_kernel<T>, grid, block, 0, s, a, interleaved));
    return OC_OK;
  }
  if (interleaved) {
    if (lpr == 8) return go(kv_append_kernel<T, 8, false>);
    if (lpr == 16) return go(kv_append_kernel<T, 16, false>);
    return go(kv_append_kernel<T, 32, false>);
  }
  if (lpr == 8) return go(kv_append_kernel<T, 8, true>);
  if (lpr == 16) return go(kv_append_kernel<T, 16, true>);
  return go(kv_append_kernel<T, 32, true>);
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
  const int64_t kd = (int64_t)c.hk * c.d, qd = (int64_t)q_heads * c.d;
  OC_REQUIRE(k_stride >= kd && v_stride >= kd && (q_heads == 0 || (q_stride >= qd && q_out_stride >= qd)),
             "kv_append: a token stride is shorter than its heads");
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
