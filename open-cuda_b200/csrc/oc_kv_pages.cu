// oc_kv_pages.cu -- bookkeeping and page moves of the paged key/value cache
// (oc_kv_cache in the public header): extend, fork, free, compact, copy.
//
// The tables live on the device, so a decode step never waits for the host.
// What has to be decided in order (which free page goes to whom) is one
// CTA's work: it reads the reference counts in page order, ranks the free
// ones with block-wide prefix sums and stops at the last page it needs, so
// the result is the same on every run and equals the sequential definition
// ("lowest free page first").  What can be done by everybody (table rows,
// counts, the pages' bytes) follows in a second kernel over the whole GPU.
// Refused calls (too few pages, an id twice) are found before anything is
// written.  Measured: room for a token of each of 64 sequences in a pool of
// 8192 pages 5 us (one CTA: four dependent trips to memory and the prefix
// sums); compaction of 266 MB over 8 layers 4.4 us of planning and 48 us of
// moves (5.5 TB/s read and written); 64 forks over 28 layers 4.3 + 15 us (their
// 16 parents' pages come from L2 for three children of four).
#include "oc_kv.cuh"

namespace oc {

constexpr int kPlanThreads = 1024;
constexpr int kScratchHead = 16;  // ints: [0] pairs to move, -1 = refused

struct KvScratch {
  int* head;
  int* list;   // [pages]    free pages in order (extend, fork); old -> new number (compact)
  int* pairs;  // [pages]    compact: sources in the first half, destinations in the second
  int* at;     // [max_seqs] first page of the list that entry i takes
};

__host__ __device__ inline KvScratch kv_scratch(int* p, int pages) {
  return KvScratch{p, p + kScratchHead, p + kScratchHead + pages, p + kScratchHead + 2 * pages + 2};
}

// The reference counts of four pages from `p` (a multiple of four); what lies
// past the pool counts as used.
__device__ __forceinline__ int4 refs4(const int* refs, int p, int pages, bool vec) {
  if (vec && p + 4 <= pages) return *reinterpret_cast<const int4*>(refs + p);
  return make_int4(p < pages ? refs[p] : 1, p + 1 < pages ? refs[p + 1] : 1, p + 2 < pages ? refs[p + 2] : 1,
                   p + 3 < pages ? refs[p + 3] : 1);
}

// The first `need` free pages, in order, into list.  Returns how many of them
// there are (block-uniform).
__device__ int find_free(const int* refs, int pages, int need, int* list, int* warp_sums) {
  const bool vec = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
  int found = 0;
  for (int p0 = 0; p0 < pages && found < need; p0 += kPlanThreads * 4) {
    const int p = p0 + threadIdx.x * 4;
    const int4 r = refs4(refs, p, pages, vec);
    const int c = (r.x <= 0) + (r.y <= 0) + (r.z <= 0) + (r.w <= 0);
    int total;
    int at = found + block_exclusive(c, warp_sums, &total);
    if (r.x <= 0 && at < need) list[at] = p;
    at += r.x <= 0;
    if (r.y <= 0 && at < need) list[at] = p + 1;
    at += r.y <= 0;
    if (r.z <= 0 && at < need) list[at] = p + 2;
    at += r.z <= 0;
    if (r.w <= 0 && at < need) list[at] = p + 3;
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

// The pages that an accepted list needs, into list; *err (shared) becomes
// kKvNoPages when there are too few.  All threads, behind a barrier that
// follows the last write to *err.  Every thread reads *err before any writes
// it again: what follows has barriers, so all have to go the same way.
__device__ __forceinline__ void plan_pages(const KvView& c, int need, int* list, int* warp_sums, int* err) {
  const bool go = *err == 0 && need > 0;
  __syncthreads();
  if (!go) return;
  const int found = need > c.pages ? 0 : find_free(c.refs, c.pages, need, list, warp_sums);
  if (found < need && threadIdx.x == 0) *err = kKvNoPages;
  __syncthreads();
}

__device__ __forceinline__ int pages_of(int tokens, int ps_shift) {
  return (int)(((int64_t)tokens + (1 << ps_shift) - 1) >> ps_shift);
}

// Marks id in a shared bitmap; true if it was marked already.
__device__ __forceinline__ bool mark(uint32_t* bits, int id) {
  const uint32_t b = 1u << (id & 31);
  return (atomicOr(&bits[id >> 5], b) & b) != 0;
}

__global__ void __launch_bounds__(kPlanThreads)
    kv_extend_kernel(KvView c, int* scratch, const int* __restrict__ seqs, const int* __restrict__ counts, int n) {
  extern __shared__ uint32_t bits[];  // [max_seqs] bits
  __shared__ int sums[33];
  __shared__ int err;
  pdl_wait();
  const KvScratch sc = kv_scratch(scratch, c.pages);
  if (threadIdx.x == 0) err = 0;
  for (int i = threadIdx.x; i < (c.max_seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  int need = 0;  // pages taken by the entries before this pass's (saturating: more than the pool is refused)
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int want = 0;
    if (i < n) {
      const int s = seqs[i], add = counts[i];
      if (s < 0 || s >= c.max_seqs || add < 0 || mark(bits, s)) {
        atomicOr(&err, kKvBadSeq);
      } else {
        const int64_t len = max(c.seq_len[s], 0), now = len + add;
        if (now > ((int64_t)c.max_pages << c.ps_shift))
          atomicOr(&err, kKvRowFull);
        else
          want = min(pages_of((int)now, c.ps_shift) - pages_of((int)len, c.ps_shift), c.pages + 1);
      }
    }
    int64_t total;
    __shared__ int64_t sums64[33];
    const int64_t before = block_exclusive<int64_t>(want, sums64, &total);
    if (i < n) sc.at[i] = (int)min((int64_t)need + before, (int64_t)c.pages);
    need = (int)min((int64_t)need + total, (int64_t)c.pages + 1);
  }
  __syncthreads();
  plan_pages(c, need, sc.list, sums, &err);
  if (err) {
    if (threadIdx.x == 0) atomicOr(c.status, err);
    return;
  }
  // a warp per entry
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {
    const int s = seqs[i];
    const int len = max(c.seq_len[s], 0), now = len + counts[i];
    const int p0 = pages_of(len, c.ps_shift), p1 = pages_of(now, c.ps_shift), at = sc.at[i];
    for (int p = p0 + lane; p < p1; p += 32) {
      const int page = sc.list[at + p - p0];
      c.table[(size_t)s * c.max_pages + p] = page;
      c.refs[page] = 1;
    }
    __syncwarp();
    if (lane == 0) c.seq_len[s] = now;
  }
}

__global__ void __launch_bounds__(kPlanThreads)
    kv_fork_plan_kernel(KvView c, int* scratch, const int* __restrict__ parents, const int* __restrict__ children,
                        int n) {
  extern __shared__ uint32_t bits[];  // [max_seqs] bits: the children
  __shared__ int sums[33];
  __shared__ int err;
  pdl_wait();
  pdl_launch();
  const KvScratch sc = kv_scratch(scratch, c.pages);
  if (threadIdx.x == 0) err = 0;
  for (int i = threadIdx.x; i < (c.max_seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = children[i];
    if (s < 0 || s >= c.max_seqs || c.seq_len[s] != 0 || mark(bits, s)) atomicOr(&err, kKvBadSeq);
  }
  __syncthreads();
  int need = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int part = 0;
    if (i < n) {
      const int s = parents[i];
      if (s < 0 || s >= c.max_seqs || ((bits[s >> 5] >> (s & 31)) & 1u)) {
        atomicOr(&err, kKvBadSeq);
      } else {
        const int len = max(c.seq_len[s], 0);
        if (pages_of(len, c.ps_shift) > c.max_pages) atomicOr(&err, kKvRowFull);
        part = (len & ((1 << c.ps_shift) - 1)) != 0;
      }
    }
    int total;
    const int before = block_exclusive(part, sums, &total);
    if (i < n) sc.at[i] = part ? need + before : -1;
    need += total;
  }
  __syncthreads();
  plan_pages(c, need, sc.list, sums, &err);
  if (threadIdx.x == 0) {
    sc.head[0] = err ? -1 : need;
    if (err) atomicOr(c.status, err);
  }
}

// Copies `bytes` (one page of one layer of one pool), all threads of the CTA.
template <typename V>
__device__ __forceinline__ void copy_block(void* dst, const void* src, size_t bytes) {
  V* d = static_cast<V*>(dst);
  const V* s = static_cast<const V*>(src);
  const int n = (int)(bytes / sizeof(V)), step = blockDim.x;
  int i = threadIdx.x;
  for (; i + 3 * step < n; i += 4 * step) {
    V x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __ldcs(s + i + j * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) __stcs(d + i + j * step, x[j]);
  }
  for (; i < n; i += step) __stcs(d + i, __ldcs(s + i));
}

// Page `from` of layer task / 2 of the keys (task even) or values to page `to`.
template <typename V>
__device__ __forceinline__ void copy_page(const KvView& c, size_t page_bytes, int task, int from, int to) {
  char* base = static_cast<char*>((task & 1) ? c.v : c.k) + (size_t)(task >> 1) * c.pages * page_bytes;
  copy_block<V>(base + (size_t)to * page_bytes, base + (size_t)from * page_bytes, page_bytes);
}

// blockIdx.x = entry, blockIdx.y = 0: its row, counts and length; 1 + task:
// its partly filled page.
template <typename V>
__global__ void __launch_bounds__(256) kv_fork_kernel(KvView c, int* scratch, const int* __restrict__ parents,
                                                      const int* __restrict__ children, size_t page_bytes) {
  pdl_wait();
  const KvScratch sc = kv_scratch(scratch, c.pages);
  if (sc.head[0] < 0) return;
  const int i = blockIdx.x, parent = parents[i], child = children[i], at = sc.at[i];
  const int len = max(c.seq_len[parent], 0), full = len >> c.ps_shift;
  const int* theirs = c.table + (size_t)parent * c.max_pages;
  if (blockIdx.y == 0) {
    int* row = c.table + (size_t)child * c.max_pages;
    for (int p = threadIdx.x; p < c.max_pages; p += blockDim.x) {
      int page = -1;
      if (p < full) {
        page = theirs[p];
        if (page >= 0 && page < c.pages)
          atomicAdd(&c.refs[page], 1);
        else
          atomicOr(c.status, kKvBadPage);
      } else if (p == full && at >= 0) {
        page = sc.list[at];
        c.refs[page] = 1;
      }
      row[p] = page;
    }
    if (threadIdx.x == 0) c.seq_len[child] = len;
  } else if (at >= 0) {
    const int from = theirs[full];
    if (from < 0 || from >= c.pages) {
      if (threadIdx.x == 0) atomicOr(c.status, kKvBadPage);
      return;
    }
    copy_page<V>(c, page_bytes, blockIdx.y - 1, from, sc.list[at]);
  }
}

// A CTA per sequence.  Each entry of the row is claimed by an exchange, so a
// sequence listed twice loses its pages once.
__global__ void __launch_bounds__(256) kv_free_kernel(KvView c, const int* __restrict__ seqs) {
  pdl_wait();
  const int s = seqs[blockIdx.x];
  if (s < 0 || s >= c.max_seqs) {
    if (threadIdx.x == 0) atomicOr(c.status, kKvBadSeq);
    return;
  }
  int* row = c.table + (size_t)s * c.max_pages;
  for (int p = threadIdx.x; p < c.max_pages; p += blockDim.x) {
    if (row[p] == -1) continue;
    const int page = atomicExch(&row[p], -1);
    if (page == -1) continue;
    if (page < 0 || page >= c.pages) {
      atomicOr(c.status, kKvBadPage);
    } else if (atomicSub(&c.refs[page], 1) <= 0) {  // nobody held it
      atomicAdd(&c.refs[page], 1);
      atomicOr(c.status, kKvBadPage);
    }
  }
  if (threadIdx.x == 0) c.seq_len[s] = 0;
}

__global__ void __launch_bounds__(kPlanThreads) kv_compact_plan_kernel(KvView c, int* scratch) {
  __shared__ int64_t sums[33];
  pdl_wait();
  pdl_launch();
  const KvScratch sc = kv_scratch(scratch, c.pages);
  const bool vec = (reinterpret_cast<uintptr_t>(c.refs) & 15) == 0;
  int live = 0;
  for (int p = threadIdx.x * 4; p < c.pages; p += kPlanThreads * 4) {
    const int4 r = refs4(c.refs, p, c.pages, vec);
    const int past = max(0, p + 4 - c.pages);  // refs4 counts those as used
    live += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0) - past;
  }
  int64_t all;
  block_exclusive<int64_t>(live, sums, &all);
  const int L = (int)all;
  // ranks of the free pages below L (low 32 bits) and of the used ones from L on
  int64_t done = 0;
  const int half = (c.pages + 1) / 2;
  for (int p0 = 0; p0 < c.pages; p0 += kPlanThreads * 4) {
    const int p = p0 + threadIdx.x * 4;
    const int4 r = refs4(c.refs, p, c.pages, vec);
    const int rr[4] = {r.x, r.y, r.z, r.w};
    int64_t mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (p + j < c.pages) mine += p + j < L ? (int64_t)(rr[j] <= 0) : (int64_t)(rr[j] > 0) << 32;
    int64_t total;
    int64_t at = done + block_exclusive(mine, sums, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p + j >= c.pages) break;
      sc.list[p + j] = p + j;
      if (p + j < L && rr[j] <= 0) {
        sc.pairs[half + (int)(at & 0xffffffff)] = p + j;
        at += 1;
      } else if (p + j >= L && rr[j] > 0) {
        sc.pairs[(int)(at >> 32)] = p + j;
        at += (int64_t)1 << 32;
      }
    }
    done += total;
  }
  __syncthreads();
  const int moves = (int)(done & 0xffffffff);
  for (int i = threadIdx.x; i < moves; i += kPlanThreads) sc.list[sc.pairs[i]] = sc.pairs[half + i];
  if (threadIdx.x == 0) sc.head[0] = moves;
}

// blockIdx.y = task (layer, keys or values); the CTAs of y = 0 also bring the
// tables and counts up to date.
template <typename V>
__global__ void __launch_bounds__(256) kv_compact_kernel(KvView c, int* scratch, size_t page_bytes) {
  pdl_wait();
  const KvScratch sc = kv_scratch(scratch, c.pages);
  const int moves = sc.head[0], half = (c.pages + 1) / 2;
  if (moves == 0) return;
  for (int i = blockIdx.x; i < moves; i += gridDim.x)
    copy_page<V>(c, page_bytes, blockIdx.y, sc.pairs[i], sc.pairs[half + i]);
  if (blockIdx.y) return;
  const size_t entries = (size_t)c.max_seqs * c.max_pages, step = (size_t)gridDim.x * blockDim.x;
  const size_t me = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (size_t e = me; e < entries; e += step) {
    const int p = c.table[e];
    if (p >= 0 && p < c.pages) {
      const int to = sc.list[p];
      if (to != p) c.table[e] = to;
    }
  }
  for (size_t i = me; i < (size_t)moves; i += step) {
    const int from = sc.pairs[i];
    c.refs[sc.pairs[half + i]] = c.refs[from];
    c.refs[from] = 0;
  }
}

// Refuses a list that writes a page twice, or writes and reads one.
__global__ void __launch_bounds__(kPlanThreads)
    kv_copy_check_kernel(KvView c, int* scratch, const int* __restrict__ src, const int* __restrict__ dst, int n) {
  extern __shared__ uint32_t bits[];  // [pages] bits: the destinations
  __shared__ int err;
  pdl_wait();
  pdl_launch();
  if (threadIdx.x == 0) err = 0;
  for (int i = threadIdx.x; i < (c.pages + 31) / 32; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= c.pages || d < 0 || d >= c.pages || mark(bits, d)) err = kKvBadPage;
  }
  __syncthreads();
  const bool in_pool = err == 0;
  __syncthreads();  // all have read it before it is written again
  if (in_pool)
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
      const int s = src[i];
      if (s != dst[i] && ((bits[s >> 5] >> (s & 31)) & 1u)) err = kKvBadPage;
    }
  __syncthreads();
  if (threadIdx.x == 0) {
    kv_scratch(scratch, c.pages).head[0] = err ? -1 : n;
    if (err) atomicOr(c.status, err);
  }
}

template <typename V>
__global__ void __launch_bounds__(256) kv_copy_kernel(KvView c, int* scratch, const int* __restrict__ src,
                                                      const int* __restrict__ dst, size_t page_bytes) {
  pdl_wait();
  if (scratch[0] < 0) return;
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  if (s != d) copy_page<V>(c, page_bytes, blockIdx.y, s, d);
}

static size_t page_bytes_of(const KvView& c, int dtype) {
  return ((size_t)c.hk << c.ps_shift) * c.d * kv_esize(dtype);
}

// Calls go(V()) with the widest type that a page's bytes and the pools'
// addresses are multiples of.
template <typename F>
static int by_width(const KvView& c, size_t page_bytes, F go) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | page_bytes;
  if (all % 16 == 0) return go(uint4());
  if (all % 4 == 0) return go(uint32_t());
  return go((unsigned short)0);
}

static int kv_pages_args(const oc_kv_cache* cache, KvView* c, int n) {
  int rc = kv_view(cache, c);
  if (rc) return rc;
  OC_REQUIRE(cache->scratch, "kv_cache: NULL scratch");
  OC_REQUIRE(c->pages <= 1 << 20 && c->max_seqs <= 1 << 18, "kv_cache: at most 2^20 pages and 2^18 sequences");
  OC_REQUIRE(c->layers <= 32767, "kv_cache: too many layers");
  OC_REQUIRE(n >= 0, "kv_cache: negative count");
  return OC_OK;
}

static int plan_smem(const void* fn, size_t bytes) {
  return smem_attr_once(fn, std::max<size_t>(bytes, 1)) ? OC_OK
                                                        : fail(OC_ERR_LAUNCH_FAILED, "kv_cache: shared memory refused");
}

}  // namespace oc

using namespace oc;

extern "C" {

int oc_kv_scratch_size(int num_pages, int max_seqs, size_t* bytes) {
  OC_REQUIRE(bytes && num_pages > 0 && max_seqs > 0 && num_pages <= 1 << 20 && max_seqs <= 1 << 18,
             "kv_cache: bad scratch shape");
  *bytes = ((size_t)kScratchHead + 2 * (size_t)num_pages + 2 + (size_t)max_seqs) * sizeof(int);
  return OC_OK;
}

int oc_kv_extend(const oc_kv_cache* cache, const int32_t* seqs, const int32_t* counts, int n, void* stream) {
  KvView c;
  if (int rc = kv_pages_args(cache, &c, n)) return rc;
  OC_REQUIRE(n <= c.max_seqs, "kv_extend: more entries than sequences");
  if (n == 0) return OC_OK;
  OC_REQUIRE(seqs && counts, "kv_extend: NULL pointer");
  const size_t smem = (size_t)(c.max_seqs + 31) / 32 * 4;
  if (int rc = plan_smem(reinterpret_cast<const void*>(kv_extend_kernel), smem)) return rc;
  OC_CHECK_CUDA(launch_pdl_ex(kv_extend_kernel, dim3(1), dim3(kPlanThreads), smem, static_cast<cudaStream_t>(stream), c,
                              cache->scratch, seqs, counts, n));
  return OC_OK;
}

int oc_kv_fork(const oc_kv_cache* cache, const int32_t* parents, const int32_t* children, int n, void* stream) {
  KvView c;
  if (int rc = kv_pages_args(cache, &c, n)) return rc;
  OC_REQUIRE(n <= c.max_seqs, "kv_fork: more entries than sequences");
  if (n == 0) return OC_OK;
  OC_REQUIRE(parents && children, "kv_fork: NULL pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t smem = (size_t)(c.max_seqs + 31) / 32 * 4, pb = page_bytes_of(c, cache->dtype);
  if (int rc = plan_smem(reinterpret_cast<const void*>(kv_fork_plan_kernel), smem)) return rc;
  OC_CHECK_CUDA(launch_pdl_ex(kv_fork_plan_kernel, dim3(1), dim3(kPlanThreads), smem, s, c, cache->scratch, parents,
                              children, n));
  return by_width(c, pb, [&](auto v) {
    OC_CHECK_CUDA(launch_pdl_ex(kv_fork_kernel<decltype(v)>, dim3(n, 1 + 2 * c.layers), dim3(256), 0, s, c,
                                cache->scratch, parents, children, pb));
    return OC_OK;
  });
}

int oc_kv_free(const oc_kv_cache* cache, const int32_t* seqs, int n, void* stream) {
  KvView c;
  if (int rc = kv_pages_args(cache, &c, n)) return rc;
  if (n == 0) return OC_OK;
  OC_REQUIRE(seqs, "kv_free: NULL pointer");
  OC_CHECK_CUDA(
      launch_pdl_ex(kv_free_kernel, dim3(n), dim3(256), 0, static_cast<cudaStream_t>(stream), c, seqs));
  return OC_OK;
}

int oc_kv_compact(const oc_kv_cache* cache, void* stream) {
  KvView c;
  if (int rc = kv_pages_args(cache, &c, 0)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t pb = page_bytes_of(c, cache->dtype);
  OC_CHECK_CUDA(launch_pdl_ex(kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, c, cache->scratch));
  // at most half of the pages move; the CTAs of a layer share what does
  const int x = std::max(1, std::min((c.pages + 1) / 2, std::max(32, std::max(1, sm_count()) * 16 / (2 * c.layers))));
  return by_width(c, pb, [&](auto v) {
    OC_CHECK_CUDA(launch_pdl_ex(kv_compact_kernel<decltype(v)>, dim3(x, 2 * c.layers), dim3(256), 0, s, c,
                                cache->scratch, pb));
    return OC_OK;
  });
}

int oc_kv_copy_pages(const oc_kv_cache* cache, const int32_t* src, const int32_t* dst, int n, void* stream) {
  KvView c;
  if (int rc = kv_pages_args(cache, &c, n)) return rc;
  OC_REQUIRE(n <= c.pages, "kv_copy_pages: more entries than pages");
  if (n == 0) return OC_OK;
  OC_REQUIRE(src && dst, "kv_copy_pages: NULL pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t smem = (size_t)(c.pages + 31) / 32 * 4, pb = page_bytes_of(c, cache->dtype);
  if (int rc = plan_smem(reinterpret_cast<const void*>(kv_copy_check_kernel), smem)) return rc;
  OC_CHECK_CUDA(launch_pdl_ex(kv_copy_check_kernel, dim3(1), dim3(kPlanThreads), smem, s, c, cache->scratch, src, dst, n));
  return by_width(c, pb, [&](auto v) {
    OC_CHECK_CUDA(launch_pdl_ex(kv_copy_kernel<decltype(v)>, dim3(n, 2 * c.layers), dim3(256), 0, s, c, cache->scratch,
                                src, dst, pb));
    return OC_OK;
  });
}

}  // extern "C"
