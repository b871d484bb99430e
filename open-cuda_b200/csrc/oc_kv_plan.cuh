// oc_kv_plan.cuh -- how attention over the paged cache is shared out.
//
// The work of a call is a list of items (sequence, kv head, block of query
// rows), each a run of key tiles; lengths differ by orders of magnitude within
// a batch and live on the device.  The tiles of all items, laid end to end,
// are cut into equal runs, one per CTA of a grid that fills the GPU once: a
// long sequence is spread over many CTAs, many short ones share a CTA, and
// nothing has to be known on the host.  A run may be as short as one tile:
// runs of two and four at least left short items waiting for one another
// (f32, 5 tokens over 40 keys, 8 heads of 128 over one: 52 us against 19).  Every CTA finds its own start with
// one block-wide prefix sum over the sequences.  An item that a cut goes
// through leaves partial results (running maximum, sum and unnormalised
// output, f32) in the workspace: a CTA has at most one item that began before
// its run (slot 0) and one that goes on after it (slot 1).  The merge kernel
// joins them in CTA order, so a call gives the same bits every time.
//
// Query rows of an item: the q_heads / kv_heads query heads of one kv head
// share its keys, so row r of a sequence and kv head is token r / G, head
// h * G + r % G: a decode step has G rows, a chunk of m tokens m * G.
#pragma once
#include "oc_kv.cuh"

namespace oc {

struct KvPlan {
  int br, bk_shift;        // query rows of an item; log2 of the keys of a tile
  int rows_min, rows_max;  // sequences with rows_min < rows <= rows_max are this launch's
  int ctas;                // grid
  int group;               // G
  uint32_t group_inv;      // floor(2^32 / G), 2^32 - 1 for 1
  int causal, window;
};

// r / G for 0 <= r < 2^31: the product with the inverse is at most one short.
__device__ __forceinline__ int plan_token(const KvPlan& p, int r) {
  int q = (int)__umulhi((uint32_t)r, p.group_inv);
  if (r - q * p.group >= p.group) ++q;
  return q;
}

// Keys [lo, hi) that rows [r0, r1] of a sequence see at all.
__device__ __forceinline__ void plan_range(const KvPlan& p, const KvSeq& s, int r0, int r1, int& lo, int& hi) {
  const int before = s.len - s.nq;
  const int first = before + plan_token(p, r0), last = before + plan_token(p, r1);
  hi = p.causal ? min(s.len, max(last + 1, 0)) : s.len;
  lo = p.window > 0 ? (int)max((int64_t)0, (int64_t)first - p.window + 1) : 0;
  lo = min(lo, hi);
}
// The same for one row.
__device__ __forceinline__ void plan_row_range(const KvPlan& p, const KvSeq& s, int r, int& lo, int& hi) {
  plan_range(p, s, r, r, lo, hi);
}

struct KvItem {
  int r0, rows;      // first row, and how many
  int lo, hi;        // keys seen by any of them
  int tile0, units;  // first tile, and how many (at least one: an item without keys still writes zeros)
};
__device__ __forceinline__ KvItem plan_item(const KvPlan& p, const KvSeq& s, int j) {
  KvItem it;
  it.r0 = j * p.br;
  it.rows = min(p.br, s.nq * p.group - it.r0);
  plan_range(p, s, it.r0, it.r0 + it.rows - 1, it.lo, it.hi);
  it.tile0 = it.lo >> p.bk_shift;
  it.units = max(1, (int)(((int64_t)it.hi + (1 << p.bk_shift) - 1) >> p.bk_shift) - it.tile0);
  return it;
}
__device__ __forceinline__ int plan_blocks(const KvPlan& p, const KvSeq& s) {
  const int rows = s.nq * p.group;
  return rows > p.rows_min && rows <= p.rows_max ? (rows + p.br - 1) / p.br : 0;
}

// A place in the list of units.
struct KvCursor {
  int b;            // entry of the batch
  KvSeq s;
  int blocks;       // row blocks of the sequence
  int h, j;         // kv head, row block
  KvItem it;
  int at;           // unit within the item
};

constexpr int kPlanSmall = 32;  // row blocks that one thread sums by itself (the threads do it side by side)

struct KvPlanShared {
  int64_t sums[33];
  int64_t off, head;
  int b, j, at, big;
};

// Units of one kv head of a sequence, by all threads of the block.
__device__ __forceinline__ int64_t plan_head_block(const KvPlan& p, const KvSeq& s, int blocks, KvPlanShared* sh) {
  int64_t u = 0, total;
  for (int j = threadIdx.x; j < blocks; j += blockDim.x) u += plan_item(p, s, j).units;
  block_exclusive<int64_t>(u, sh->sums, &total);
  return total;
}

// Sets the cursor to unit index * chunk.  Returns the number of units that
// exist (0: none at or after that place); *chunk is the length of a run.
// Block-wide: all threads call it with the same arguments and leave with the
// same cursor.  A thread sums the sequences that are its own; sequences of
// many row blocks (a chunk of 2048 tokens has hundreds) are summed by all.
// The CTA of index 0, which sees every entry, reports those with new tokens
// whose id is outside the table.
__device__ __forceinline__ int64_t plan_locate(const KvPlan& p, const KvView& c, const KvBatch& bt, int index,
                                               KvPlanShared* sh, int64_t* chunk, KvCursor& cur) {
  if (bt.n == 1) {  // one sequence of few row blocks: every thread sees all there is
    const KvSeq s = kv_seq(c, bt, 0);
    const int blocks = plan_blocks(p, s);
    if (blocks == 0) return 0;
    if (index == 0 && s.s < 0) atomicOr(c.status, kKvBadSeq);
    if (blocks <= 8) {
      int64_t head = 0;
      for (int j = 0; j < blocks; ++j) head += plan_item(p, s, j).units;
      const int64_t all = head * c.hk;
      *chunk = (all + p.ctas - 1) / p.ctas;
      int64_t off = *chunk * index;
      if (off >= all) return 0;
      cur.b = 0;
      cur.s = s;
      cur.blocks = blocks;
      cur.h = (int)(off / head);
      off -= cur.h * head;
      for (cur.j = 0;; ++cur.j) {
        cur.it = plan_item(p, s, cur.j);
        if (off < cur.it.units) break;
        off -= cur.it.units;
      }
      cur.at = (int)off;
      return all;
    }
  }
  int64_t total = 0, u;
  bool have = false;
  if (threadIdx.x == 0) sh->b = -1;
  // the units of the sequences, blockDim at a time: the sum first, then (a
  // second round) the place; one round does both when it sees all sequences
  const bool once = bt.n <= (int)blockDim.x;
  for (int round = once ? 1 : 0; round < 2; ++round) {
    if (round == 1 && !once) {
      *chunk = (total + p.ctas - 1) / p.ctas;
      u = *chunk * index;
      if (u >= total) return 0;
      have = true;
    }
    int64_t done = 0;
    for (int b0 = 0; b0 < bt.n; b0 += blockDim.x) {
      const int b = b0 + threadIdx.x;
      KvSeq s{-1, 0, 0, 0};
      if (b < bt.n) s = kv_seq(c, bt, b);
      const int blocks = plan_blocks(p, s);
      if (index == 0 && blocks > 0 && s.s < 0) atomicOr(c.status, kKvBadSeq);
      int64_t head = 0;
      if (blocks <= kPlanSmall)
        for (int j = 0; j < blocks; ++j) head += plan_item(p, s, j).units;
      if (__syncthreads_or(blocks > kPlanSmall)) {
        // one after another, in order: the next one is the lowest left
        int left = blocks > kPlanSmall;
        for (;;) {
          if (threadIdx.x == 0) sh->big = INT_MAX;
          __syncthreads();
          if (left) atomicMin(&sh->big, b);
          __syncthreads();
          const int big = sh->big;
          if (big == INT_MAX) break;
          const KvSeq t = kv_seq(c, bt, big);
          const int64_t sum = plan_head_block(p, t, plan_blocks(p, t), sh);
          if (b == big) head = sum, left = 0;
        }
      }
      int64_t sum;
      const int64_t before = done + block_exclusive<int64_t>(head * c.hk, sh->sums, &sum);
      done += sum;
      if (once) {
        *chunk = (done + p.ctas - 1) / p.ctas;
        u = *chunk * index;
        if (u >= done) return 0;
        have = true;
      }
      if (have && before <= u && u < before + head * c.hk) sh->b = b, sh->off = u - before, sh->head = head;
      __syncthreads();
      if (have && sh->b >= 0) break;
    }
    total = once || round == 0 ? done : total;
  }
  cur.b = sh->b;
  cur.s = kv_seq(c, bt, cur.b);
  cur.blocks = plan_blocks(p, cur.s);
  int64_t off = sh->off;
  if (cur.blocks == 1) {
    cur.h = (int)(off / sh->head);
    cur.j = 0;
    cur.it = plan_item(p, cur.s, 0);
    cur.at = (int)(off - cur.h * sh->head);
    return total;
  }
  cur.h = (int)(off / sh->head);
  off -= cur.h * sh->head;
  int64_t before = 0;
  for (int j0 = 0;; j0 += blockDim.x) {
    const int j = j0 + threadIdx.x;
    const int64_t w = j < cur.blocks ? plan_item(p, cur.s, j).units : 0;
    int64_t sum;
    const int64_t mine = before + block_exclusive<int64_t>(w, sh->sums, &sum);
    if (mine <= off && off < mine + w) sh->j = j, sh->at = (int)(off - mine);
    before += sum;
    if (off < before || j0 + (int)blockDim.x >= cur.blocks) break;
  }
  __syncthreads();
  cur.j = sh->j;
  cur.at = sh->at;
  cur.it = plan_item(p, cur.s, cur.j);
  return total;
}

// The next item's first unit; false at the end of the list.  Whole warps.
__device__ __forceinline__ bool plan_next(const KvPlan& p, const KvView& c, const KvBatch& bt, KvCursor& cur) {
  cur.at = 0;
  if (++cur.j >= cur.blocks) {
    cur.j = 0;
    if (++cur.h >= c.hk) {
      cur.h = 0;
      // 32 entries at a time: thousands of the other class may lie between
      const int lane = threadIdx.x & 31;
      if (++cur.b >= bt.n) return false;
      cur.s = kv_seq(c, bt, cur.b);
      cur.blocks = plan_blocks(p, cur.s);
      for (int b0 = cur.b + 1; cur.blocks == 0; b0 += 32) {
        if (b0 >= bt.n) return false;
        const int b = b0 + lane;
        const uint32_t some = __ballot_sync(0xffffffffu, b < bt.n && plan_blocks(p, kv_seq(c, bt, b)) > 0);
        if (some) {
          cur.b = b0 + __ffs(some) - 1;
          cur.s = kv_seq(c, bt, cur.b);
          cur.blocks = plan_blocks(p, cur.s);
        }
      }
    }
  }
  cur.it = plan_item(p, cur.s, cur.j);
  return true;
}

// What the cut behind a CTA's run goes through, and whether a result of the
// run's whole items is not finite, for the merge kernel.
struct KvCut {
  int pieces, lost;  // (read as a pair) 0: nothing
  int b, h, r0, rows, q0, unused;
};

// Partial results of CTA `cta`, slot 0 or 1: m [br], l [br], o [br][dp]
// (16-byte aligned), f32;
// in front of them the cuts, one per CTA.
__host__ __device__ inline size_t plan_slot_o(int br) { return (2 * (size_t)br + 3) / 4 * 4; }  // where o begins
__host__ __device__ inline size_t plan_slot_floats(int br, int dp) { return plan_slot_o(br) + (size_t)br * dp; }
__host__ __device__ inline size_t plan_cut_floats(int ctas) { return (size_t)ctas * (sizeof(KvCut) / sizeof(float)); }

struct KvAttn {
  KvView c;
  KvBatch bt;
  KvPlan p;
  size_t layer_off;  // elements before the layer in each pool
  const void* q;
  void* out;
  int64_t qs, os;
  float scale2;  // scale * log2(e)
  int vec;       // rows of the pools are whole 16-byte chunks
  int qvec;      // rows of q are
  int ovec16;    // rows of out are whole 16-byte chunks
  int ovec;      // pairs of elements of out are 4-byte aligned
  int beside;    // follows a launch of the same call, and may run beside it
  float* ws;
  int* dev_status;
};

__device__ __forceinline__ float* plan_slot(const KvAttn& a, int cta, int slot, int dp) {
  return a.ws + plan_cut_floats(a.p.ctas) + ((size_t)cta * 2 + slot) * plan_slot_floats(a.p.br, dp);
}

// One thread of a CTA: what its run leaves to the CTAs behind it.
__device__ __forceinline__ void plan_no_cut(const KvAttn& a) {
  KvCut& cut = reinterpret_cast<KvCut*>(a.ws)[blockIdx.x];
  cut.pieces = cut.lost = 0;
}
// The last item of its run began there and goes on: rest = its units behind the run.
__device__ __forceinline__ void plan_cut(const KvAttn& a, const KvCursor& cur, int rest, int64_t chunk) {
  KvCut& cut = reinterpret_cast<KvCut*>(a.ws)[blockIdx.x];
  cut.b = cur.b, cut.h = cur.h, cut.r0 = cur.it.r0, cut.rows = cur.it.rows, cut.q0 = cur.s.q0;
  cut.pieces = 2 + (int)((rest - 1) / chunk);
}
// One thread: a result of the run's whole items is not finite.
__device__ __forceinline__ void plan_lost(const KvAttn& a) { reinterpret_cast<KvCut*>(a.ws)[blockIdx.x].lost = 1; }

constexpr int kMostCtas = 2048;  // of an attention kernel's grid

// The partial results of one launch.
struct KvPart {
  float* ws;
  int ctas, br, groups, dp;  // groups: of R rows, that an item can have; dp: floats of a row
  KvPlan p;
};
struct KvParts {
  KvPart of[2];
  int count;
};

// Joins the partial results of a call's launches, and computes again what they
// lost (oc_kv_merge.cu).  few: one row of an item at a time; dp: the widest.
int kv_merge(const KvAttn& a, const KvParts& parts, int dtype, bool few, int dp, int grid, cudaStream_t s);

}  // namespace oc
