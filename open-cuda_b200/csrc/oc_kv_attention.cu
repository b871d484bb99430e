// oc_kv_attention.cu -- oc_kv_attention: new tokens attend to their
// sequences' pages (oc_kv_plan.cuh says how the work is shared out).
#include <map>

#include "oc_kv_plan.cuh"
#include "oc_kv_tile32.cuh"

namespace oc {

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
    e = std::min(std::max(1, per) * std::max(1, sm_count()), kMostCtas);
  }
  return e;
}

// One launch over a class of the batch's sequences: the kernel, its shape.
struct KvLaunch {
  void (*kern)(KvAttn) = nullptr;
  void (*tile)(KvAttn, CUtensorMap, CUtensorMap, CUtensorMap, int, int) = nullptr;  // or this one
  const void* fn() const { return kern ? reinterpret_cast<const void*>(kern) : reinterpret_cast<const void*>(tile); }
  int br = 0, bk = 0, dp = 0, threads = 0;
  int rows_min = 0, rows_max = INT_MAX;
  size_t smem = 0;
  int ctas = 0;
  bool one_per_sm = false;  // it takes all of an SM's tensor memory
  int merge_rows = 0;  // rows that an item of a call can have
};

template <typename K>
static KvLaunch shape_of(void (*kern)(KvAttn)) {
  KvLaunch l;
  l.kern = kern;
  l.br = K::ROWS, l.bk = K::BK, l.dp = K::DP, l.threads = K::THREADS, l.smem = K::SMEM;
  return l;
}

// On the CUDA cores; `rows`: the most that a sequence's kv head can have.
// The rows of an item are the registers' and the multiply-adds' cost, used or
// not: one token over 20000 keys, 32 f32 heads of 128 over 8, takes 72 us in
// items of 4 rows (2.3 TB/s) and 153 in items of 8.  (What bounds it:
// oc_kv_rows.cuh.)
template <typename T>
static KvLaunch scalar_launch(int d, int rows) {
  auto go = [](auto k) { return shape_of<decltype(k)>(kv_rows_kernel<decltype(k)>); };
  if constexpr (sizeof(T) == 4) {
    if (d <= 64) return rows <= 1 ? go(KvRows<T, 64, 1>()) : rows <= 4 ? go(KvRows<T, 64, 4>()) : go(KvRows<T, 64, 8>());
    if (d <= 128) return rows <= 1 ? go(KvRows<T, 128, 1>()) : rows <= 4 ? go(KvRows<T, 128, 4>()) : go(KvRows<T, 128, 8>());
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
  auto go = [](auto k) { return shape_of<decltype(k)>(kv_mma_kernel<decltype(k)>); };
  if (d <= 64) return rows <= 16 ? go(KvMma<T, 64, 1>()) : go(KvMma<T, 64, 2>());
  if (d <= 96) return rows <= 16 ? go(KvMma<T, 96, 1>()) : go(KvMma<T, 96, 2>());
  if (d <= 128) return rows <= 16 ? go(KvMma<T, 128, 1>()) : go(KvMma<T, 128, 2>());
  return go(KvMma<T, 256, 1>());
}

// Rows of the pools are whole, aligned 16-byte chunks.
static bool vector_rows(const KvView& c, size_t esize) { return c.d * esize % 16 == 0 && aligned16(c.k) && aligned16(c.v); }

// Query rows of a sequence's kv head up to which the few-row kernels take it
// where both can.  Measured, 128-row tiles against them: f16, 16 sequences of
// 4096 keys and heads of 128, 16 rows 103 us : 87, 28 rows 103 : 114, 64 rows
// 106 : 179; one sequence of 16000, 16 rows 48 : 32, 28 rows 50 : 56.  f32, 16
// of 4000 and heads of 64, 8 rows 245 : 238, 16 rows 257 : 453; one sequence,
// 8 rows 36 : 36, 16 rows 38 : 48.
template <typename T>
constexpr int kFewRows = sizeof(T) == 4 ? 8 : 16;

// The launches of a call, each over its class of sequences.  one_each: every
// sequence has one new token; qvec: rows of q are whole 16-byte chunks.
template <typename T>
static int pick(const KvView& c, int tokens, int n, int q_heads, bool one_each, bool qvec, KvLaunch (&out)[2]) {
  const int group = q_heads / c.hk;
  const int most = one_each ? group : tokens * group;                 // rows that a sequence can have
  const int likely = tokens <= n ? std::min(group, most) : most;      // and those to choose a shape by
  constexpr int few = kFewRows<T>;
  const bool tile = c.d <= 128 && likely > few && is_sm100() && (sizeof(T) == 4 || (qvec && vector_rows(c, sizeof(T))));
  int count = 0;
  if (!tile) {
    if constexpr (sizeof(T) == 4)
      out[count++] = scalar_launch<T>(c.d, likely);
    else
      out[count++] = vector_rows(c, sizeof(T)) ? mma_launch<T>(c.d, likely) : scalar_launch<T>(c.d, likely);
  } else {
    if (group <= few) {  // else a single token has more rows
      if constexpr (sizeof(T) == 4) {
        // beside long chunks the few rows are mostly single tokens', unless the
        // whole batch is of a few tokens each
        const int64_t mean = (int64_t)tokens * group / std::max(1, n);
        out[count] = scalar_launch<T>(c.d, mean <= 4 * few ? few : group);
      } else {
        out[count] = mma_launch<T>(c.d, few);
      }
      out[count++].rows_max = few;
    }
    if constexpr (sizeof(T) == 4) {
      auto go = [](auto k) { return shape_of<decltype(k)>(kv_tile32_kernel<decltype(k)>); };
      out[count] = c.d <= 64 ? go(KvTile32<64>()) : go(KvTile32<128>());
    } else {
      auto go = [](auto k) {
        KvLaunch l = shape_of<decltype(k)>(nullptr);
        l.tile = kv_tile_kernel<decltype(k)>;
        return l;
      };
      out[count] = c.d <= 64 ? go(KvTile<T, 64>()) : go(KvTile<T, 128>());
    }
    out[count].rows_min = count ? few : 0;
    out[count++].one_per_sm = true;
  }
  for (int i = 0; i < count; ++i) {
    const void* fn = out[i].fn();
    smem_attr_once(fn, out[i].smem);  // before the occupancy is asked for
    out[i].ctas = out[i].one_per_sm ? std::max(1, sm_count()) : resident_ctas(fn, out[i].threads, out[i].smem);
    out[i].merge_rows = std::min(out[i].br, std::min(most, out[i].rows_max));
  }
  return count;
}

// Each launch has a part of the workspace (16-byte aligned: slots are).
static size_t part_floats(const KvLaunch& l) {
  return plan_cut_floats(l.ctas) + (size_t)l.ctas * 2 * plan_slot_floats(l.br, l.dp);
}
static size_t workspace_floats(const KvLaunch* l, int count) {
  size_t sum = 0;
  for (int i = 0; i < count; ++i) sum += part_floats(l[i]);
  return sum;
}

template <typename T>
static int run(KvAttn a, int q_heads, bool one_each, void* ws, size_t ws_bytes, cudaStream_t s) {
  KvLaunch l[2];
  const int count = pick<T>(a.c, a.bt.total, a.bt.n, q_heads, one_each, a.qvec, l);
  OC_REQUIRE(ws && aligned16(ws) && ws_bytes >= workspace_floats(l, count) * sizeof(float),
             "kv_attention: workspace too small or not 16-byte aligned");
  KvParts parts = {};
  a.ws = static_cast<float*>(ws);
  int dp = 0, rows = 0;
  for (int i = 0; i < count; ++i) {
    a.p.br = l[i].br, a.p.bk_shift = __builtin_ctz(l[i].bk), a.p.rows_min = l[i].rows_min, a.p.rows_max = l[i].rows_max;
    a.p.ctas = l[i].ctas;
    a.beside = i > 0;
    if (!smem_attr_once(l[i].fn(), l[i].smem)) return fail(OC_ERR_LAUNCH_FAILED, "kv_attention: shared memory attribute refused");
    const dim3 grid(l[i].ctas), block(l[i].threads);
    if (l[i].kern) {
      OC_CHECK_CUDA(launch_pdl_ex(l[i].kern, grid, block, l[i].smem, s, a));
    } else {
      // the pools as matrices of head_dim columns; a box is a page, or a tile of a larger one
      const KvView& c = a.c;
      const uint64_t pool_rows = ((uint64_t)c.layers * c.pages * c.hk) << c.ps_shift;
      const int box = c.ps_shift < 3 || pool_rows > INT_MAX ? 0 : std::min(1 << c.ps_shift, l[i].bk);
      const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
      CUtensorMap m[3] = {};
      for (int x = 0; box && x < 2; ++x)
        if (int rc = make_tmap_2d(&m[x], x ? c.v : c.k, type, sizeof(T), c.d, pool_rows, (uint64_t)c.d * sizeof(T), 64, box,
                                  CU_TENSOR_MAP_SWIZZLE_128B))
          return rc;
      // the queries as [token][head][feature]: a box is all heads of a group, of 128 / G tokens
      const int g = a.p.group, qbox = 128 % g == 0 ? 128 / g : 0;
      if (qbox)
        if (int rc = make_tmap_3d(&m[2], a.q, type, c.d, q_heads, (uint64_t)c.d * sizeof(T), a.bt.total, (uint64_t)a.qs * sizeof(T), 64, g,
                                  qbox, CU_TENSOR_MAP_SWIZZLE_128B))
          return rc;
      OC_CHECK_CUDA(launch_pdl_ex(l[i].tile, grid, block, l[i].smem, s, a, m[0], m[1], m[2], box, qbox));
    }
    parts.of[i] = KvPart{a.ws, l[i].ctas, l[i].br, 0, l[i].dp, a.p};
    a.ws += part_floats(l[i]);
    dp = std::max(dp, l[i].dp);
    rows = std::max(rows, l[i].merge_rows);
  }
  // the rows of one item that the joining kernel takes at a time: see there
  const bool few = count == 1 && rows <= 16;
  int64_t tasks = 0;
  parts.count = count;
  for (int i = 0; i < count; ++i) {
    parts.of[i].groups = few ? l[i].merge_rows : (l[i].merge_rows + 7) / 8;
    tasks += (int64_t)(l[i].ctas - 1) * parts.of[i].groups;
  }
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(tasks, (few ? 4 : 8) * (int64_t)std::max(1, sm_count())));
  return kv_merge(a, parts, sizeof(T) == 4 ? OC_KV_F32 : std::is_same<T, __half>::value ? OC_KV_F16 : OC_KV_BF16, few, dp, grid, s);
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
  size_t most = 0;
  for (int form = 0; form < 4; ++form) {  // whatever cu and the alignment of q will be
    KvLaunch l[2];
    const bool one_each = form & 1, qvec = form & 2;
    const int count = cache->dtype == OC_KV_F32   ? pick<float>(c, tokens, n, q_heads, one_each, qvec, l)
                      : cache->dtype == OC_KV_F16 ? pick<__half>(c, tokens, n, q_heads, one_each, qvec, l)
                                                  : pick<__nv_bfloat16>(c, tokens, n, q_heads, one_each, qvec, l);
    most = std::max(most, workspace_floats(l, count));
  }
  *bytes = most * sizeof(float);
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
  OC_REQUIRE(!kv_overlap(q, q_stride * es, qd * es, out, out_stride * es, qd * es, tokens), "kv_attention: out overlaps q");  // rows may be computed twice
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
  a.ovec16 = c.d * es % 16 == 0 && aligned16(out) && out_stride * es % 16 == 0;
  a.ovec = c.d % 2 == 0 && reinterpret_cast<uintptr_t>(out) % (2 * es) == 0 && out_stride % 2 == 0;
  a.ws = nullptr;
  a.dev_status = device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->dtype == OC_KV_F32) return run<float>(a, q_heads, cu == nullptr, workspace, workspace_bytes, s);
  if (cache->dtype == OC_KV_F16) return run<__half>(a, q_heads, cu == nullptr, workspace, workspace_bytes, s);
  return run<__nv_bfloat16>(a, q_heads, cu == nullptr, workspace, workspace_bytes, s);
}

}  // extern "C"
