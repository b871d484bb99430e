// oc_kv_plan.cuh -- how attention over the paged cache is shared out.
//
// The work of a call is a list of items (sequence, kv head, block of query
// rows), each a run of key tiles; lengths differ by orders of magnitude within
// a batch and live on the device.  The tiles of all items, laid end to end,
// are cut into equal runs, one per CTA of a grid that fills the GPU once: a
// long sequence is spread over many CTAs, many short ones share a CTA, and
// nothing has to be known on the host.  Every CTA finds its own start with
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
  int br, bk;              // query rows of an item, keys of a tile
  int rows_min, rows_max;  // sequences with rows_min < rows <= rows_max are this launch's
  int ctas, min_units;     // grid, and the shortest run worth a CTA of its own
  int group;               // G
  int causal, window;
};

// Keys [lo, hi) that rows [r0, r1] of a sequence see at all.
__device__ __forceinline__ void plan_range(const KvPlan& p, const KvSeq& s, int r0, int r1, int& lo, int& hi) {
  const int before = s.len - s.nq;
  const int first = before + r0 / p.group, last = before + r1 / p.group;
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
  it.tile0 = it.lo / p.bk;
  it.units = max(1, (int)(((int64_t)it.hi + p.bk - 1) / p.bk) - it.tile0);
  return it;
}
__device__ __forceinline__ int plan_blocks(const KvPlan& p, const KvSeq& s) {
  const int rows = s.nq * p.group;
  return rows > p.rows_min && rows <= p.rows_max ? (rows + p.br - 1) / p.br : 0;
}
// Units of one kv head of a sequence.
__device__ __forceinline__ int64_t plan_head_units(const KvPlan& p, const KvSeq& s) {
  int64_t u = 0;
  const int nb = plan_blocks(p, s);
  for (int j = 0; j < nb; ++j) u += plan_item(p, s, j).units;
  return u;
}

// A place in the list of units.
struct KvCursor {
  int b;            // entry of the batch
  KvSeq s;
  int64_t head;     // units of one of its kv heads
  int h, j;         // kv head, row block
  KvItem it;
  int at;           // unit within the item
};

struct KvPlanShared {
  int64_t sums[33];
  int64_t off;
  int b;
};

// Sets the cursor to unit index * chunk.  Returns the number of units that
// exist (0: none at or after that place); *chunk is the length of a run.
// Block-wide: all threads call it with the same arguments and leave with the
// same cursor.
__device__ __forceinline__ int64_t plan_locate(const KvPlan& p, const KvView& c, const KvBatch& bt, int index,
                                               KvPlanShared* sh, int64_t* chunk, KvCursor& cur) {
  const int per = (bt.n + blockDim.x - 1) / blockDim.x;
  const int b0 = min(bt.n, (int)threadIdx.x * per), b1 = min(bt.n, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += plan_head_units(p, kv_seq(c, bt, b)) * c.hk;
  int64_t total;
  int64_t before = block_exclusive<int64_t>(mine, sh->sums, &total);
  const int64_t run = max((int64_t)p.min_units, (total + p.ctas - 1) / p.ctas);
  *chunk = run;
  const int64_t u = run * index;
  if (u >= total) return 0;
  if (before <= u && u < before + mine) {
    for (int b = b0; b < b1; ++b) {
      const int64_t w = plan_head_units(p, kv_seq(c, bt, b)) * c.hk;
      if (u < before + w) {
        sh->b = b;
        sh->off = u - before;
        break;
      }
      before += w;
    }
  }
  __syncthreads();
  cur.b = sh->b;
  cur.s = kv_seq(c, bt, cur.b);
  cur.head = plan_head_units(p, cur.s);
  int64_t off = sh->off;
  cur.h = (int)(off / cur.head);
  off -= cur.h * cur.head;
  cur.j = 0;
  for (;;) {
    cur.it = plan_item(p, cur.s, cur.j);
    if (off < cur.it.units) break;
    off -= cur.it.units;
    ++cur.j;
  }
  cur.at = (int)off;
  return total;
}

// The next item's first unit; false at the end of the list.
__device__ __forceinline__ bool plan_next(const KvPlan& p, const KvView& c, const KvBatch& bt, KvCursor& cur) {
  cur.at = 0;
  if (++cur.j >= plan_blocks(p, cur.s)) {
    cur.j = 0;
    if (++cur.h >= c.hk) {
      cur.h = 0;
      for (;;) {
        if (++cur.b >= bt.n) return false;
        cur.s = kv_seq(c, bt, cur.b);
        if (plan_blocks(p, cur.s) > 0) break;
      }
    }
  }
  cur.it = plan_item(p, cur.s, cur.j);
  return true;
}

// Partial results of CTA `cta`, slot 0 or 1: m [br], l [br], o [br][dp], f32.
__host__ __device__ inline size_t plan_slot_floats(int br, int dp) { return (size_t)br * (dp + 2); }

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
  int ovec;      // pairs of elements of out are 4-byte aligned
  float* ws;
  int* dev_status;
};

__device__ __forceinline__ float* plan_slot(const KvAttn& a, int cta, int slot, int dp) {
  return a.ws + ((size_t)cta * 2 + slot) * plan_slot_floats(a.p.br, dp);
}

}  // namespace oc
