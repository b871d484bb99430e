// oc_kv_merge.cu -- the last kernel of an attention call over the paged cache:
// joins the pieces of the items that cuts went through (oc_kv_plan.cuh), and
// computes the rows whose result is not finite again, from the definition.
//
// Such rows come from values that a row does not see (a weight of 0 does not
// hide an infinity or a NaN), from sums that overflow where their mean does
// not, and from f32 values that two f16 terms do not hold (oc_kv_tile32.cuh).
// They are rare, and this is the place for them: nothing waits for this
// kernel, and the whole GPU is free to take them.
#include "oc_kv_rows.cuh"

namespace oc {

// One row of one query head from the definition, by all threads of a block
// (whole warps): for rows whose result was lost.  Reads only keys that the row
// sees, each once: a warp takes 32 of them at a time and keeps what it has so
// far divided by the sum so far, so that values near the type's largest do not
// overflow (the fast kernels divide at the end); the warps meet in `sh`
// (kv_exact_floats).
template <typename T, int DP>
__device__ __noinline__ void kv_row_exact(const KvAttn& a, KvSeq s, int h, int row, float* sh) {
  const KvView& c = a.c;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = c.d, g = a.p.group;
  const int64_t token = s.q0 + row / g, head = (int64_t)(h * g + row % g) * d;
  const T* q = static_cast<const T*>(a.q) + token * a.qs + head;
  const T* kb = static_cast<const T*>(c.k) + a.layer_off;
  const T* vb = static_cast<const T*>(c.v) + a.layer_off;
  int lo, hi;
  plan_row_range(a.p, s, row, lo, hi);
  constexpr int NF = DP / 32, U = 2;  // features a lane, keys in flight
  float x[NF], o[NF] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < NF; ++i) x[i] = lane + 32 * i < d ? kv_f32(q[lane + 32 * i]) : 0.0f;
  for (int64_t key0 = lo + 32 * (int64_t)warp; key0 < hi; key0 += 32 * warps) {
    const int n = (int)min((int64_t)32, hi - key0);
    const int64_t off = kv_row_off(a, s.s, h, (int)(key0 + min(lane, n - 1)), lo, hi);  // -1: a bad page, keys and values of zero
    float score = -INFINITY;
    for (int j0 = 0; j0 < n; j0 += U) {
      float dot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = __shfl_sync(0xffffffffu, off, min(j0 + u, n - 1));
        dot[u] = 0.0f;
#pragma unroll
        for (int i = 0; i < NF; ++i)
          if (lane + 32 * i < d && at >= 0) dot[u] = fmaf(x[i], kv_f32(kb[at + lane + 32 * i]), dot[u]);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], w);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lane == j0 + u && lane < n) score = dot[u] * a.scale2;
    }
    float mn = score;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
    mn = fmaxf(m, mn);
    const float base = mn == -INFINITY ? 0.0f : mn, p = lane < n ? exp2f(score - base) : 0.0f;
    float ln = p;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) ln += __shfl_xor_sync(0xffffffffu, ln, w);
    const float before = l * exp2f(m - base);
    l = before + ln;
    m = mn;
    const float keep = l == 0.0f ? 0.0f : before / l, weight = l == 0.0f ? 0.0f : p / l;
#pragma unroll
    for (int i = 0; i < NF; ++i) o[i] *= keep;
#pragma unroll 2
    for (int j = 0; j < n; ++j) {
      const int64_t at = __shfl_sync(0xffffffffu, off, j);
      const float w = __shfl_sync(0xffffffffu, weight, j);
#pragma unroll
      for (int i = 0; i < NF; ++i)
        if (lane + 32 * i < d && at >= 0) o[i] = fmaf(w, kv_f32(vb[at + lane + 32 * i]), o[i]);
    }
  }
  float *ms = sh + warps * d, *ls = ms + warps;
#pragma unroll
  for (int i = 0; i < NF; ++i)
    if (lane + 32 * i < d) sh[warp * d + lane + 32 * i] = o[i];
  if (lane == 0) ms[warp] = m, ls[warp] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < warps; ++w) top = fmaxf(top, ms[w]);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int w = 0; w < warps; ++w) sum = fmaf(ls[w], exp2f(ms[w] - base), sum);
  T* out = static_cast<T*>(a.out) + token * a.os + head;
  for (int e = threadIdx.x; e < d; e += blockDim.x) {
    float y = 0.0f;
    for (int w = 0; w < warps; ++w) y = fmaf(ls[w] * exp2f(ms[w] - base) / sum, sh[w * d + e], y);
    out[e] = kv_from<T>(sum == 0.0f ? 0.0f : y);
  }
  __syncthreads();
}
// Floats of `sh` for d features.
constexpr int kv_exact_floats(int threads, int d) { return threads / 32 * (d + 2); }

// Whether the row holds a result that is not finite.
template <typename T>
__device__ __forceinline__ bool kv_row_lost(const KvAttn& a, const KvSeq& s, int h, int row, int first, int step) {
  const int g = a.p.group, d = a.c.d;
  const T* out = static_cast<const T*>(a.out) + (int64_t)(s.q0 + row / g) * a.os + (int64_t)(h * g + row % g) * d;
  bool lost = false;
  for (int e = first; e < d; e += step) lost |= !isfinite(kv_f32(out[e]));
  return lost;
}

// Rows whose result is not finite, from the definition (oc_kv_rows.cuh): those
// of this merge CTA's tasks, and its share of those that the attention kernels
// left in their whole items.  All threads of the CTA.
template <typename T, int R, int DP>
__device__ __noinline__ void kv_merge_exact(const KvAttn& a, const KvParts& parts, unsigned short* list0, const unsigned short* list1,
                                            int tasks0, int tasks, float* meet) {
  __shared__ KvPlanShared plan;
  auto row = [&](KvSeq s, int h, int r) {
    if (__syncthreads_or(kv_row_lost<T>(a, s, h, r, threadIdx.x, blockDim.x))) kv_row_exact<T, DP>(a, s, h, r, meet);
  };
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const bool second = task >= tasks0;
    const KvPart& pt = parts.of[second];
    const int number = second ? task - tasks0 : task;
    const KvCut cut = reinterpret_cast<const KvCut*>(pt.ws)[(second ? list1 : list0)[number / pt.groups]];
    const KvSeq s = kv_seq(a.c, a.bt, cut.b);
    const int r0 = number % pt.groups * R, r1 = min(cut.rows, r0 + R);
    for (int r = r0; r < r1; ++r) row(s, cut.h, cut.r0 + r);
  }
  for (int k = 0; k < parts.count; ++k) {
    const KvPart& pt = parts.of[k];
    // the attention CTAs that lost some, in order
    int found = 0;
    for (int c0 = 0; c0 < pt.ctas; c0 += blockDim.x) {
      const int cta = c0 + threadIdx.x;
      const int lost = cta < pt.ctas && reinterpret_cast<const KvCut*>(pt.ws)[cta].lost;
      int64_t sum;
      const int at = found + (int)block_exclusive<int64_t>(lost, plan.sums, &sum);
      if (lost) list0[at] = (unsigned short)cta;
      found += (int)sum;
    }
    __syncthreads();
    // each one's rows are shared by as many CTAs as there are for it
    const int shares = max(1, (int)gridDim.x / max(1, found));
    for (int job = blockIdx.x; job < found * shares; job += gridDim.x) {
      const int cta = list0[job % found], share = job / found;
      KvCursor cur;
      int64_t chunk;
      const int64_t total = plan_locate(pt.p, a.c, a.bt, cta, &plan, &chunk, cur);
      for (int64_t left = min(chunk, total - chunk * cta); left > 0;) {
        const int t1 = (int)min((int64_t)cur.it.units, cur.at + left);
        if (cur.at == 0 && t1 == cur.it.units)
          for (int r = share; r < cur.it.rows; r += shares) row(cur.s, cur.h, cur.it.r0 + r);
        left -= t1 - cur.at;
        if (left > 0) plan_next(pt.p, a.c, a.bt, cur);
      }
      __syncthreads();  // (plan_locate's shared memory)
    }
    __syncthreads();
  }
}

// Joins the pieces of the items that cuts went through.  R rows of an item at
// a time: one, its pieces shared by the 8 warps, for decode steps, where an
// item of a long sequence has few rows and dozens of pieces; eight, a warp
// each, for chunks, whose items have many rows and two or three pieces.  The
// outputs are requested together with the maxima they are weighted by, so a
// row costs one trip to memory.  Every CTA lists the cuts that went through
// an item and takes its share of their rows: a CTA per possible cut and row
// would mostly be launched to find nothing (2065 CTAs, 8 us, at 296 x 7).
// DP: features of a row, 128 or 256.
template <typename T, int R, int DP>
__global__ void __launch_bounds__(256, R == 1 ? 2 : 4) kv_merge_kernel(const __grid_constant__ KvAttn a, const __grid_constant__ KvParts parts) {
  constexpr int WARPS = 8, SPLIT = WARPS / R, NV = DP / 128;  // warps that share a row
  __shared__ alignas(16) float meet[kv_exact_floats(32 * WARPS, DP)];  // R == 1: rows of outputs, written four features at a time, maxima and sums
  float(*part)[DP] = reinterpret_cast<float(*)[DP]>(meet);
  float *ms = meet + WARPS * DP, *ls = ms + WARPS;
  __shared__ unsigned short list[2][kMostCtas];
  __shared__ int wcount[2][WARPS];
  const KvView& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = c.d;
  pdl_wait();
  // each thread looks at every 256th CTA's cut, all requested at once; the
  // order of the list does not matter
  constexpr int ROUNDS = kMostCtas / 256;
  uint32_t mine[2] = {0, 0};
  int lost = 0;  // a result that is not finite
  int before[2], found[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k < parts.count) {
      const KvCut* cuts = reinterpret_cast<const KvCut*>(parts.of[k].ws);
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const int cta = i * 256 + threadIdx.x;
        if (cta < parts.of[k].ctas) {
          const int2 x = *reinterpret_cast<const int2*>(&cuts[cta]);  // pieces, lost
          if (x.x > 0) mine[k] |= 1u << i;
          lost |= x.y;
        }
      }
    }
    before[k] = __popc(mine[k]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before[k], o);
      if (lane >= o) before[k] += y;
    }
    if (lane == 31) wcount[k][warp] = before[k];
    before[k] -= __popc(mine[k]);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before[k] += wcount[k][w];
      found[k] += wcount[k][w];
    }
    for (uint32_t todo = mine[k]; todo; todo &= todo - 1) list[k][before[k]++] = (unsigned short)((__ffs(todo) - 1) * 256 + threadIdx.x);
  }
  __syncthreads();
  const int tasks0 = found[0] * parts.of[0].groups, tasks = tasks0 + found[1] * parts.of[1].groups;
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const bool second = task >= tasks0;
    const KvPart& pt = parts.of[second];
    const int number = second ? task - tasks0 : task, br = pt.br, dp = pt.dp;
    const int cta = list[second][number / pt.groups];
    const KvCut cut = reinterpret_cast<const KvCut*>(pt.ws)[cta];
    const int pieces = cut.pieces, r = (number % pt.groups) * R + warp / SPLIT;
    if (r >= cut.rows) continue;  // R == 1: the whole CTA; else the warp has nobody to meet
    const size_t slot = plan_slot_floats(br, dp), step = 2 * slot;
    // piece 0 is in slot 1 of that CTA, piece i in slot 0 of the i-th behind it
    const float* first = pt.ws + plan_cut_floats(pt.ctas) + (size_t)cta * step + slot;
    const float* rest = first + slot;
    constexpr int U = R == 1 ? 8 : 2;
    float m = -INFINITY, l = 0.0f;
    float4 acc[NV] = {};  // features 4 lane .. (and 128 + 4 lane ..)
    for (int i0 = warp % SPLIT; i0 < pieces; i0 += SPLIT * U) {
      float pm[U], pl[U];
      float4 po[U][NV];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * SPLIT;
        pm[u] = -INFINITY, pl[u] = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) po[u][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < pieces) {
          const float* s = i == 0 ? first : rest + (size_t)(i - 1) * step;
          const float* o = s + plan_slot_o(br) + (size_t)r * dp;
          pm[u] = s[r];
          pl[u] = s[br + r];
#pragma unroll
          for (int k = 0; k < NV; ++k)
            if (128 * k + 4 * lane < dp) po[u][k] = *reinterpret_cast<const float4*>(o + 128 * k + 4 * lane);
        }
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, pm[u]);
      const float base = mn == -INFINITY ? 0.0f : mn, corr = exp2f(m - base);
      m = mn;
      l *= corr;
#pragma unroll
      for (int k = 0; k < NV; ++k) acc[k].x *= corr, acc[k].y *= corr, acc[k].z *= corr, acc[k].w *= corr;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = exp2f(pm[u] - base);
        l = fmaf(w, pl[u], l);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          acc[k].x = fmaf(w, po[u][k].x, acc[k].x);
          acc[k].y = fmaf(w, po[u][k].y, acc[k].y);
          acc[k].z = fmaf(w, po[u][k].z, acc[k].z);
          acc[k].w = fmaf(w, po[u][k].w, acc[k].w);
        }
      }
    }
    const int rr = cut.r0 + r, token = plan_token(a.p, rr);
    T* out = static_cast<T*>(a.out) + (int64_t)(cut.q0 + token) * a.os + (int64_t)(cut.h * a.p.group + rr - token * a.p.group) * d;
    if constexpr (R == 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k) *reinterpret_cast<float4*>(&part[warp][128 * k + 4 * lane]) = acc[k];
      if (lane == 0) ms[warp] = m, ls[warp] = l;
      __syncthreads();
      float mm = ms[0];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) mm = fmaxf(mm, ms[k]);
      const float base = mm == -INFINITY ? 0.0f : mm;
      if ((int)threadIdx.x < d) {
        float sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
          const float w = exp2f(ms[k] - base);
          sum = fmaf(w, ls[k], sum);
          o = fmaf(w, part[k][threadIdx.x], o);
        }
        o = sum == 0.0f ? 0.0f : o / sum;
        out[threadIdx.x] = kv_from<T>(o);
        lost |= kv_lost<T>(o);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const float f[4] = {acc[k].x, acc[k].y, acc[k].z, acc[k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = 128 * k + 4 * lane + e;
          if (x < d) {
            const float o = l == 0.0f ? 0.0f : f[e] / l;
            out[x] = kv_from<T>(o);
            lost |= kv_lost<T>(o);
          }
        }
      }
    }
  }
  if (__syncthreads_or(lost)) kv_merge_exact<T, R, DP>(a, parts, list[0], list[1], tasks0, tasks, meet);
}

int kv_merge(const KvAttn& a, const KvParts& parts, int dtype, bool few, int dp, int grid, cudaStream_t s) {
  auto by_type = [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kern) {
      OC_CHECK_CUDA(launch_pdl_ex(kern, dim3(grid), dim3(256), 0, s, a, parts));
      return OC_OK;
    };
    if (dp <= 128) return few ? go(kv_merge_kernel<T, 1, 128>) : go(kv_merge_kernel<T, 8, 128>);
    return few ? go(kv_merge_kernel<T, 1, 256>) : go(kv_merge_kernel<T, 8, 256>);
  };
  if (dtype == OC_KV_F32) return by_type(float());
  if (dtype == OC_KV_F16) return by_type(__half());
  return by_type(__nv_bfloat16());
}

}  // namespace oc
