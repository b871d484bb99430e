"""Paged key/value cache on the CUDA library: many sequences' keys and values
in pages, the operators that fill, read and manage them.

The reference keeps one growing Vec per head (KvCacheHead,
crates/open-cuda-llm/src/lib.rs:530-596), one sequence at a time.  Here
sequences of any length share one pool of pages, all tables live on the
device, and no call waits for the host, so a decode step of many sequences
can be captured into a CUDA graph.

    cache = KVCache.create(layers, pages, page_size, kv_heads, head_dim, torch.bfloat16, max_seqs, max_pages_per_seq)
    cache.extend(seqs, counts)                       # room for the new tokens
    for layer in range(layers):
        q = cache.append(layer, q, k, v, cu, seqs, q_weight=qw, k_weight=kw, inv_freq=inv)
        o = cache.attention(layer, q, cu, seqs)
    cache.fork(parents, children); cache.free(seqs); cache.compact()
    cache.check()                                    # raises if a call was refused on the device

`seqs`, `counts`, `cu`, ... are int32 CUDA tensors: entry b of a batch is
sequence seqs[b] (seqs None: b) with new tokens cu[b] .. cu[b + 1] - 1 (cu
None: one token each).  Calls on one cache are ordered by the caller (one
stream, or events); attention alone may run on several streams at once.
"""
from __future__ import annotations

import ctypes as C
import math

import opencuda_cuda as oc

NO_PAGES, BAD_SEQUENCE, ROW_FULL, BAD_PAGE = 1, 2, 4, 8
_REASONS = {NO_PAGES: "too few free pages", BAD_SEQUENCE: "a sequence id outside the table, used twice, or a child that is not empty",
            ROW_FULL: "more tokens than a row of the page table holds", BAD_PAGE: "a page number outside the pool, or a token without a page"}


class _Cache(C.Structure):
    """oc_kv_cache of the public header."""

    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("page_table", C.c_void_p), ("seq_len", C.c_void_p), ("refcount", C.c_void_p),
                ("status", C.c_void_p), ("scratch", C.c_void_p), ("dtype", C.c_int), ("num_layers", C.c_int), ("num_pages", C.c_int),
                ("kv_heads", C.c_int), ("page_size", C.c_int), ("head_dim", C.c_int), ("max_seqs", C.c_int), ("max_pages_per_seq", C.c_int)]


class KVCache:
    """A cache over the caller's tensors (see create for new ones).

    k, v        [layers, pages, kv_heads, page_size, head_dim], f32, f16 or bf16
    page_table  [max_seqs, max_pages_per_seq] int32, -1 where there is no page
    seq_len     [max_seqs] int32; refcount [pages] int32; status [1] int32"""

    def __init__(self, k, v, page_table, seq_len, refcount, status=None):
        torch = oc._torch()
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("kv_cache: k and v are [layers, pages, kv_heads, page_size, head_dim] of one type")
        dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        if k.dtype not in dtypes:
            raise ValueError(f"kv_cache: {k.dtype} is not float32, float16 or bfloat16")
        if page_table.dim() != 2 or seq_len.shape != (page_table.shape[0],) or refcount.shape != (k.shape[1],):
            raise ValueError("kv_cache: page_table [max_seqs, max_pages_per_seq], seq_len [max_seqs], refcount [pages]")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=k.device)
        for t in (page_table, seq_len, refcount, status):
            if t.dtype != torch.int32:
                raise ValueError("kv_cache: the tables are int32")
        for t in (k, v, page_table, seq_len, refcount, status):
            oc._need_cuda(t)
            if not t.is_contiguous() or t.device != k.device:
                raise ValueError("kv_cache: contiguous tensors on one device expected")
        layers, pages, heads, page_size, dim = k.shape
        need = oc.sz(0)
        oc.check(oc.lib().oc_kv_scratch_size(pages, page_table.shape[0], C.byref(need)))
        self.k, self.v, self.page_table, self.seq_len, self.refcount, self.status = k, v, page_table, seq_len, refcount, status
        self.scratch = torch.empty(need.value // 4, dtype=torch.int32, device=k.device)
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = layers, pages, heads, page_size, dim
        self.dtype, self.device = k.dtype, k.device
        self._c = _Cache(k.data_ptr(), v.data_ptr(), page_table.data_ptr(), seq_len.data_ptr(), refcount.data_ptr(), status.data_ptr(),
                         self.scratch.data_ptr(), dtypes[k.dtype], layers, pages, heads, page_size, dim, *page_table.shape)
        self._p = C.byref(self._c)
        self._index = k.device.index
        self._int32 = torch.int32
        self._cuda = torch.cuda
        self._empty = torch.empty
        self._ws_bytes = {}
        ws = oc.sz(0)
        oc.check(oc.lib().oc_kv_attention_workspace_size(self._p, 0, 0, heads, C.byref(ws)))  # checks the shape as a whole

    @classmethod
    def create(cls, layers, pages, page_size, kv_heads, head_dim, dtype, max_seqs, max_pages_per_seq, device="cuda"):
        """A fresh, empty cache."""
        torch = oc._torch()
        shape = (layers, pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.full((max_seqs, max_pages_per_seq), -1, dtype=torch.int32, device=device),
                   torch.zeros(max_seqs, dtype=torch.int32, device=device), torch.zeros(pages, dtype=torch.int32, device=device))

    # -- argument checks --

    def _ids(self, t, what):
        if t.dtype != self._int32 or t.dim() != 1 or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"kv_cache: {what} is a contiguous int32 vector on {self.device}")
        return t.numel()

    def _batch(self, tokens, cu, seqs):
        if cu is None:
            n = tokens
        else:
            n = self._ids(cu, "cu") - 1
            if n < 0:
                raise ValueError("kv_cache: cu holds one number more than there are sequences")
        if seqs is not None and self._ids(seqs, "seqs") != n:
            raise ValueError(f"kv_cache: {seqs.numel()} sequences for {n} entries")
        return n

    def _rows(self, t, heads, what):
        """Token stride of a [tokens, heads, head_dim] tensor whose tokens are contiguous."""
        if t.dim() != 3 or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"kv_cache: {what} is [tokens, {'heads' if heads is None else heads}, {self.head_dim}], got {tuple(t.shape)}")
        if t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"kv_cache: {what} is {self.dtype} on {self.device}")
        st = t.stride()
        if (t.shape[2] > 1 and st[2] != 1) or (t.shape[1] > 1 and st[1] != self.head_dim):
            raise ValueError(f"kv_cache: the heads of a token of {what} must be contiguous")
        return max(st[0], t.shape[1] * self.head_dim) if t.shape[0] <= 1 else st[0]

    def _call(self, fn, *args):
        """Calls fn on the cache's device and that device's current stream."""
        if self._cuda.current_device() == self._index:
            oc.check(fn(self._p, *args, self._cuda.current_stream().cuda_stream))
        else:
            with self._cuda.device(self._index):
                oc.check(fn(self._p, *args, self._cuda.current_stream().cuda_stream))

    # -- bookkeeping --

    def extend(self, seqs, counts):
        """Sequence seqs[i] grows by counts[i] tokens; the pages it lacks are
        taken from the free ones, lowest number first."""
        n = self._ids(seqs, "seqs")
        if self._ids(counts, "counts") != n:
            raise ValueError("kv_cache: one count per sequence")
        self._call(oc.lib().oc_kv_extend, seqs.data_ptr(), counts.data_ptr(), n)

    def fork(self, parents, children):
        """children[i] (empty) becomes a copy of parents[i]: full pages are
        shared, a partly filled last page is copied over all layers."""
        n = self._ids(parents, "parents")
        if self._ids(children, "children") != n:
            raise ValueError("kv_cache: one parent per child")
        self._call(oc.lib().oc_kv_fork, parents.data_ptr(), children.data_ptr(), n)

    def free(self, seqs):
        """The sequences give their pages back."""
        n = self._ids(seqs, "seqs")
        self._call(oc.lib().oc_kv_free, seqs.data_ptr(), n)

    def compact(self):
        """Moves the pages in use to the pool's front."""
        self._call(oc.lib().oc_kv_compact)

    def copy_pages(self, src, dst):
        """Page dst[i] := page src[i] over all layers; tables and counts stay."""
        n = self._ids(src, "src")
        if self._ids(dst, "dst") != n:
            raise ValueError("kv_cache: one destination per source")
        self._call(oc.lib().oc_kv_copy_pages, src.data_ptr(), dst.data_ptr(), n)

    def check(self):
        """Waits for the cache's device and raises ValueError if a call since
        the last check met something it refuses."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise ValueError("kv_cache: " + "; ".join(text for bit, text in _REASONS.items() if bits & bit))

    # -- a layer's tokens --

    def append(self, layer, q, k, v, cu=None, seqs=None, q_weight=None, k_weight=None, eps=1e-6, inv_freq=None, interleaved=False,
               q_out=None):
        """Norms (q_weight, k_weight [head_dim]) and rotation (inv_freq
        [rot_dim / 2] f32) of the new tokens' queries [tokens, q_heads,
        head_dim] and keys [tokens, kv_heads, head_dim], keys and values
        written to their pages.  Returns the queries (q_out, or a new tensor;
        q None: keys and values alone)."""
        ks, vs = self._rows(k, self.kv_heads, "k"), self._rows(v, self.kv_heads, "v")
        tokens = k.shape[0]
        n = self._batch(tokens, cu, seqs)
        heads = qs = os_ = qp = op = 0
        if q is not None:
            qs, heads = self._rows(q, None, "q"), q.shape[1]
            if q_out is None:
                q_out = self._empty(q.shape, dtype=self.dtype, device=self.device)
            os_ = self._rows(q_out, heads, "q_out")
            if q.shape[0] != tokens or q_out.shape[0] != tokens:
                raise ValueError("kv_cache: q, k, v and q_out have the same tokens")
            qp, op = q.data_ptr(), q_out.data_ptr()
        if v.shape[0] != tokens:
            raise ValueError("kv_cache: q, k, v and q_out have the same tokens")
        wp = []
        for w in (q_weight, k_weight):
            if w is not None and (w.shape != (self.head_dim,) or w.dtype != self.dtype or not w.is_contiguous() or w.device != self.device):
                raise ValueError(f"kv_cache: a norm's weight is [{self.head_dim}] {self.dtype} on {self.device}")
            wp.append(None if w is None else w.data_ptr())
        rot, ip = 0, None
        if inv_freq is not None:
            if inv_freq.dim() != 1 or str(inv_freq.dtype) != "torch.float32" or not inv_freq.is_contiguous() or inv_freq.device != self.device:
                raise ValueError(f"kv_cache: inv_freq is a float32 vector on {self.device}")
            rot, ip = 2 * inv_freq.shape[0], inv_freq.data_ptr()
        self._call(oc.lib().oc_kv_append, layer, tokens, n, None if cu is None else cu.data_ptr(), None if seqs is None else seqs.data_ptr(),
                   heads, qp, qs, k.data_ptr(), ks, v.data_ptr(), vs, op, os_, wp[0], wp[1], eps, ip, rot, int(interleaved))
        return q_out

    def attention(self, layer, q, cu=None, seqs=None, scale=None, causal=True, window=0, out=None):
        """softmax(scale q . K^T) V of the new tokens' queries [tokens,
        q_heads, head_dim] over their sequences' pages (scale None: 1 /
        sqrt(head_dim)); causal, and the last `window` keys alone when window
        > 0.  Rows of `out` behind the last sequence stay as they are."""
        qs = self._rows(q, None, "q")
        tokens, heads, d = q.shape
        n = self._batch(tokens, cu, seqs)
        if out is None:
            out = self._empty(q.shape, dtype=self.dtype, device=self.device)
        elif out.shape[0] != tokens:
            raise ValueError("kv_cache: out has q's shape")
        os_ = self._rows(out, heads, "out")
        key = (tokens, n, heads)
        need = self._ws_bytes.get(key)
        if need is None:
            size = oc.sz(0)
            with self._cuda.device(self._index):
                oc.check(oc.lib().oc_kv_attention_workspace_size(self._p, tokens, n, heads, C.byref(size)))
            if len(self._ws_bytes) > 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[key] = max(16, size.value)
        ws = self._empty(need, dtype=self._torch_uint8, device=self.device)
        self._call(oc.lib().oc_kv_attention, layer, tokens, n, None if cu is None else cu.data_ptr(), None if seqs is None else seqs.data_ptr(),
                   heads, q.data_ptr(), qs, out.data_ptr(), os_, 1.0 / math.sqrt(d) if scale is None else scale, int(bool(causal)), window,
                   ws.data_ptr(), need)
        return out

    @property
    def _torch_uint8(self):
        return oc._torch().uint8
