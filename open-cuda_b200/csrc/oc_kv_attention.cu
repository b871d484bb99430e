// oc_kv_attention.cu -- oc_kv_attention: new tokens attend to their
// sequences' pages (oc_kv_plan.cuh says how the work is shared out).
#include <map>

#include "oc_kv_plan.cuh"
#include "oc_kv_mma.cuh"

namespace oc {

// Joins the pieces of one item that a cut went through: blockIdx.x = the CTA
// whose run it began in, blockIdx.y = the row.
template <typename T>
__global__ void __launch_bounds__(128) kv_merge_kernel(KvAttn a, int dp) {
  __shared__ float part[4][256], lsum[4];
  const KvView& c = a.c;
  pdl_wait();
  const KvCut cut = reinterpret_cast<const KvCut*>(a.ws)[blockIdx.x];
  const int r = blockIdx.y, pieces = cut.pieces;
  if (pieces == 0 || r >= cut.rows) return;
  const size_t step = 2 * plan_slot_floats(a.p.br, dp);
  // piece 0 is in slot 1 of that CTA, piece i in slot 0 of the i-th behind it
  const float* first = plan_slot(a, blockIdx.x, 1, dp);
  const float* rest = plan_slot(a, blockIdx.x + 1, 0, dp);
  auto at = [&](int i) { return i == 0 ? first : rest + (size_t)(i - 1) * step; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, br = a.p.br, d = c.d;
  float m = -INFINITY;
  for (int i = lane; i < pieces; i += 32) m = fmaxf(m, at(i)[r]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float acc[8] = {};
#pragma unroll 4
  for (int i = warp; i < pieces; i += 4) {
    const float* s = at(i);
    const float w = exp2f(s[r] - base);
    l = fmaf(w, s[br + r], l);
    const float* o = s + 2 * br + (size_t)r * dp;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < d) acc[e] = fmaf(w, o[lane + 32 * e], acc[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[warp][lane + 32 * e] = acc[e];
  if (lane == 0) lsum[warp] = l;
  __syncthreads();
  const float ls = lsum[0] + lsum[1] + lsum[2] + lsum[3];
  const int rr = cut.r0 + r, g = a.p.group;
  T* out = static_cast<T*>(a.out) + (int64_t)(cut.q0 + rr / g) * a.os + (int64_t)(cut.h * g + rr % g) * d;
  bool bad = false;
  for (int e = threadIdx.x; e < d; e += blockDim.x) {
    const float o = ls == 0.0f ? 0.0f : (part[0][e] + part[1][e] + part[2][e] + part[3][e]) / ls;
    out[e] = kv_from<T>(o);
    bad |= !isfinite(o);
  }
  // (oc_kv_mma.cuh) a row that is not finite is computed from the definition
  if (__syncthreads_or(bad) && warp == 0) kv_row_exact<T>(a, kv_seq(c, a.bt, cut.b), cut.h, rr);
}

// CTAs of a kernel that fit the GPU at once, remembered per device and kernel.
static int resident_ctas(const void* fn, int threads, size_t smem) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  auto& e = known[std::make_pair(dev, fn)];
  if (e == 0) {
    int per = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, fn, threads, smem) != cudaSuccess) {
      cudaGetLastError();
      per = 0;
    }
    e = std::max(1, per) * std::max(1, sm_count());
  }
  return e;
}

// One launch over a class of the batch's sequences: the kernel, its shape.
struct KvLaunch {
  void (*kern)(KvAttn) = nullptr;
  int br = 0, bk = 0, dp = 0, threads = 0, min_units = 1;
  int rows_min = 0, rows_max = INT_MAX;
  size_t smem = 0;
  int ctas = 0;
  int merge_rows = 0;  // rows that an item of a call can have
};

template <typename K>
static KvLaunch shape_of(void (*kern)(KvAttn), int min_units) {
  KvLaunch l;
  l.kern = kern;
  l.br = K::ROWS, l.bk = K::BK, l.dp = K::DP, l.threads = K::THREADS, l.min_units = min_units, l.smem = K::SMEM;
  return l;
}

// On the CUDA cores; `rows`: the most that a sequence's kv head can have.
template <typename T>
static KvLaunch scalar_launch(int d, int rows) {
  auto go = [](auto k) { return shape_of<decltype(k)>(kv_rows_kernel<decltype(k)>, 4); };
  if constexpr (sizeof(T) == 4) {
    if (d <= 64) return rows <= 1 ? go(KvRows<T, 64, 1>()) : go(KvRows<T, 64, 8>());
    if (d <= 128) return rows <= 1 ? go(KvRows<T, 128, 1>()) : go(KvRows<T, 128, 8>());
    return go(KvRows<T, 256, 4>());
  } else {
    if (d <= 64) return go(KvRows<T, 64, 4>());
    if (d <= 128) return go(KvRows<T, 128, 4>());
    return go(KvRows<T, 256, 4>());
  }
}

// On warp-level matrix instructions.
template <typename T>
static KvLaunch mma_launch(int d, int rows) {
  auto go = [](auto k) { return shape_of<decltype(k)>(kv_mma_kernel<decltype(k)>, 2); };
  if (d <= 64) return rows <= 16 ? go(KvMma<T, 64, 1>()) : go(KvMma<T, 64, 2>());
  if (d <= 96) return rows <= 16 ? go(KvMma<T, 96, 1>()) : go(KvMma<T, 96, 2>());
  if (d <= 128) return rows <= 16 ? go(KvMma<T, 128, 1>()) : go(KvMma<T, 128, 2>());
  return go(KvMma<T, 256, 1>());
}

// Rows of the pools are whole, aligned 16-byte chunks.
static bool vector_rows(const KvView& c, size_t esize) { return c.d * esize % 16 == 0 && aligned16(c.k) && aligned16(c.v); }

// The launches of a call, each over its class of sequences.
template <typename T>
static int pick(const KvView& c, int tokens, int n, int q_heads, KvLaunch (&out)[2]) {
  const int group = q_heads / c.hk;
  const int rows = tokens <= n ? group : INT_MAX;
  if constexpr (sizeof(T) == 2) {
    out[0] = vector_rows(c, sizeof(T)) ? mma_launch<T>(c.d, rows) : scalar_launch<T>(c.d, rows);
  } else {
    out[0] = scalar_launch<T>(c.d, rows);
  }
  const int count = 1;
  for (int i = 0; i < count; ++i) {
    const void* fn = reinterpret_cast<const void*>(out[i].kern);
    smem_attr_once(fn, out[i].smem);  // before the occupancy is asked for
    out[i].ctas = resident_ctas(fn, out[i].threads, out[i].smem);
    out[i].merge_rows = std::min(out[i].br, rows);
  }
  return count;
}

static size_t workspace_floats(const KvLaunch* l, int count) {
  size_t most = 0;
  for (int i = 0; i < count; ++i) most = std::max(most, plan_cut_floats(l[i].ctas) + (size_t)l[i].ctas * 2 * plan_slot_floats(l[i].br, l[i].dp));
  return most;
}

template <typename T>
static int run(KvAttn a, int q_heads, void* ws, size_t ws_bytes, cudaStream_t s) {
  KvLaunch l[2];
  const int count = pick<T>(a.c, a.bt.total, a.bt.n, q_heads, l);
  OC_REQUIRE(ws && aligned16(ws) && ws_bytes >= workspace_floats(l, count) * sizeof(float),
             "kv_attention: workspace too small or not 16-byte aligned");
  for (int i = 0; i < count; ++i) {
    a.p.br = l[i].br, a.p.bk_shift = __builtin_ctz(l[i].bk), a.p.rows_min = l[i].rows_min, a.p.rows_max = l[i].rows_max;
    a.p.ctas = l[i].ctas, a.p.min_units = l[i].min_units;
    a.ws = static_cast<float*>(ws);
    if (!smem_attr_once(reinterpret_cast<const void*>(l[i].kern), l[i].smem))
      return fail(OC_ERR_LAUNCH_FAILED, "kv_attention: shared memory attribute refused");
    OC_CHECK_CUDA(launch_pdl_ex(l[i].kern, dim3(l[i].ctas), dim3(l[i].threads), l[i].smem, s, a));
    if (l[i].ctas > 1)
      OC_CHECK_CUDA(launch_pdl_ex(kv_merge_kernel<T>, dim3(l[i].ctas - 1, l[i].merge_rows), dim3(128), 0, s, a, l[i].dp));
  }
  return OC_OK;
}

static int attn_args(const oc_kv_cache* cache, KvView* c, int tokens, int n, int q_heads) {
  if (int rc = kv_view(cache, c)) return rc;
  OC_REQUIRE(tokens >= 0 && n >= 0, "kv_attention: negative size");
  OC_REQUIRE(q_heads > 0 && q_heads % c->hk == 0, "kv_attention: q_heads must be a multiple of kv_heads");
  OC_REQUIRE((int64_t)tokens * q_heads <= INT_MAX, "kv_attention: too many query rows");
  return OC_OK;
}

}  // namespace oc

using namespace oc;

extern "C" {

int oc_kv_attention_workspace_size(const oc_kv_cache* cache, int tokens, int n, int q_heads, size_t* bytes) {
  KvView c;
  if (int rc = attn_args(cache, &c, tokens, n, q_heads)) return rc;
  OC_REQUIRE(bytes, "kv_attention: NULL pointer");
  KvLaunch l[2];
  const int count = cache->dtype == OC_KV_F32   ? pick<float>(c, tokens, n, q_heads, l)
                    : cache->dtype == OC_KV_F16 ? pick<__half>(c, tokens, n, q_heads, l)
                                                : pick<__nv_bfloat16>(c, tokens, n, q_heads, l);
  *bytes = workspace_floats(l, count) * sizeof(float);
  return OC_OK;
}

int oc_kv_attention(const oc_kv_cache* cache, int layer, int tokens, int n, const int32_t* cu, const int32_t* seqs,
                    int q_heads, const void* q, int64_t q_stride, void* out, int64_t out_stride, float scale,
                    int causal, int window, void* workspace, size_t workspace_bytes, void* stream) {
  KvView c;
  if (int rc = attn_args(cache, &c, tokens, n, q_heads)) return rc;
  OC_REQUIRE(layer >= 0 && layer < c.layers, "kv_attention: no such layer");
  OC_REQUIRE(cu || n == tokens, "kv_attention: without cu each sequence has one token");
  OC_REQUIRE(window >= 0, "kv_attention: negative window");
  if (tokens == 0 || n == 0) return OC_OK;
  OC_REQUIRE(q && out, "kv_attention: NULL pointer");
  const int64_t qd = (int64_t)q_heads * c.d;
  OC_REQUIRE(q_stride >= qd && out_stride >= qd, "kv_attention: a token stride is shorter than its heads");
  const size_t es = kv_esize(cache->dtype);
  KvAttn a;
  a.c = c;
  a.bt = KvBatch{cu, seqs, n, tokens};
  a.p = KvPlan{};
  a.p.group = q_heads / c.hk;
  a.p.group_inv = a.p.group == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / a.p.group);
  a.p.causal = causal != 0;
  a.p.window = window;
  a.layer_off = (((size_t)layer * c.pages * c.hk) << c.ps_shift) * c.d;
  a.q = q, a.out = out, a.qs = q_stride, a.os = out_stride;
  a.scale2 = scale * 1.44269504088896341f;
  a.vec = vector_rows(c, es);
  a.qvec = c.d * es % 16 == 0 && aligned16(q) && q_stride * es % 16 == 0;
  a.ovec = c.d % 2 == 0 && reinterpret_cast<uintptr_t>(out) % (2 * es) == 0 && out_stride % 2 == 0;
  a.ws = nullptr;
  a.dev_status = device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->dtype == OC_KV_F32) return run<float>(a, q_heads, workspace, workspace_bytes, s);
  if (cache->dtype == OC_KV_F16) return run<__half>(a, q_heads, workspace, workspace_bytes, s);
  return run<__nv_bfloat16>(a, q_heads, workspace, workspace_bytes, s);
}

}  // extern "C"
