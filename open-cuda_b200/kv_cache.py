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
stream, or events); attention alone may run on several streams and from
several threads at once.
"""
from __future__ import annotations

import ctypes as C
import math
import threading

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
        # what every call needs: one attribute away
        lib = oc.lib()
        self._torch, self._index, self._int32, self._f32 = torch, k.device.index, torch.int32, torch.float32
        self._current_device, self._raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        self._capturing, self._empty_like, self._scale = torch.cuda.is_current_stream_capturing, torch.empty_like, 1.0 / math.sqrt(dim)
        self._append, self._attention, self._extend, self._fork = lib.oc_kv_append, lib.oc_kv_attention, lib.oc_kv_extend, lib.oc_kv_fork
        self._free, self._compact, self._copy = lib.oc_kv_free, lib.oc_kv_compact, lib.oc_kv_copy_pages
        self._ws_bytes, self._workspaces, self._turn = {}, {}, threading.Lock()
        ws = oc.sz(0)
        oc.check(lib.oc_kv_attention_workspace_size(self._p, 0, 0, heads, C.byref(ws)))  # checks the shape as a whole

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
        """Entries of the batch, and the addresses of cu and seqs."""
        if cu is None:
            n, cp = tokens, None
        else:
            n, cp = self._ids(cu, "cu") - 1, cu.data_ptr()
            if n < 0:
                raise ValueError("kv_cache: cu holds one number more than there are sequences")
        if seqs is None:
            return n, cp, None
        if self._ids(seqs, "seqs") != n:
            raise ValueError(f"kv_cache: {seqs.numel()} sequences for {n} entries")
        return n, cp, seqs.data_ptr()

    def _rows(self, t, tokens, heads, what):
        """Token stride of a [tokens, heads, head_dim] tensor whose tokens are contiguous."""
        shape, d = t.shape, self.head_dim
        if len(shape) != 3 or shape[0] != tokens or shape[1] != heads or shape[2] != d:
            raise ValueError(f"kv_cache: {what} is [{tokens}, {heads}, {d}], got {tuple(shape)}")
        if t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"kv_cache: {what} is {self.dtype} on {self.device}")
        s0, s1, s2 = t.stride()
        if (s2 != 1 and d > 1) or (s1 != d and heads > 1):
            raise ValueError(f"kv_cache: the heads of a token of {what} must be contiguous")
        return s0 if tokens > 1 else max(s0, heads * d)

    def _call(self, fn, *args):
        """Calls fn on the cache's device and that device's current stream."""
        index = self._index
        if self._current_device() == index:
            rc = fn(self._p, *args, self._raw_stream(index))
        else:
            with self._torch.cuda.device(index):
                rc = fn(self._p, *args, self._raw_stream(index))
        if rc:
            oc.check(rc)

    def _new_bytes(self, need):
        return self._torch.empty(need, dtype=self._torch.uint8, device=self.device)

    # -- bookkeeping --

    def extend(self, seqs, counts):
        """Sequence seqs[i] grows by counts[i] tokens; the pages it lacks are
        taken from the free ones, lowest number first."""
        n = self._ids(seqs, "seqs")
        if self._ids(counts, "counts") != n:
            raise ValueError("kv_cache: one count per sequence")
        self._call(self._extend, seqs.data_ptr(), counts.data_ptr(), n)

    def fork(self, parents, children):
        """children[i] (empty) becomes a copy of parents[i]: full pages are
        shared, a partly filled last page is copied over all layers."""
        n = self._ids(parents, "parents")
        if self._ids(children, "children") != n:
            raise ValueError("kv_cache: one parent per child")
        self._call(self._fork, parents.data_ptr(), children.data_ptr(), n)

    def free(self, seqs):
        """The sequences give their pages back."""
        n = self._ids(seqs, "seqs")
        self._call(self._free, seqs.data_ptr(), n)

    def compact(self):
        """Moves the pages in use to the pool's front."""
        self._call(self._compact)

    def copy_pages(self, src, dst):
        """Page dst[i] := page src[i] over all layers; tables and counts stay."""
        n = self._ids(src, "src")
        if self._ids(dst, "dst") != n:
            raise ValueError("kv_cache: one destination per source")
        self._call(self._copy, src.data_ptr(), dst.data_ptr(), n)

    def check(self):
        """Waits for the cache's device and raises ValueError if a call since
        the last check met something it refuses, OcError if a wait inside a
        kernel expired."""
        self._torch.cuda.synchronize(self.device)  # calls of every stream
        bits = int(self.status.item())
        expired = oc.ci(0)
        with self._torch.cuda.device(self._index):
            oc.check(oc.lib().oc_get_device_status(C.byref(expired)))
        if expired.value:
            raise oc.OcError(oc.OC_ERR_TIMEOUT, f"kv_cache: a wait inside a kernel expired (code {expired.value})")
        if bits:
            self.status.zero_()
            raise ValueError("kv_cache: " + "; ".join(text for bit, text in _REASONS.items() if bits & bit))

    # -- a layer's tokens --

    def append(self, layer, q, k, v, cu=None, seqs=None, q_weight=None, k_weight=None, eps=1e-6, inv_freq=None, interleaved=False,
               q_out=None):
        """Norms (q_weight, k_weight [head_dim]) and rotation (inv_freq
        [rot_dim / 2] f32) of the new tokens' queries [tokens, q_heads,
        head_dim] and keys [tokens, kv_heads, head_dim], keys and values
        written to their pages.  Returns the queries (q_out, or a new tensor,
        unset behind the last sequence; q None: keys and values alone)."""
        index = self._index
        if self._current_device() != index:
            with self._torch.cuda.device(index):
                return self.append(layer, q, k, v, cu, seqs, q_weight, k_weight, eps, inv_freq, interleaved, q_out)
        tokens, d = k.shape[0], self.head_dim
        ks, vs = self._rows(k, tokens, self.kv_heads, "k"), self._rows(v, tokens, self.kv_heads, "v")
        n, cp, sp = self._batch(tokens, cu, seqs)
        heads = qs = os_ = 0
        qp = op = None
        if q is not None:
            heads = q.shape[1]
            qs = self._rows(q, tokens, heads, "q")
            if q_out is None:
                q_out = self._empty_like(q)  # contiguous: the heads of q's tokens are
                os_ = heads * d
            else:
                os_ = self._rows(q_out, tokens, heads, "q_out")
            qp, op = q.data_ptr(), q_out.data_ptr()
        qw = kw = ip = None
        rot = 0
        if q_weight is not None:
            qw = self._weight(q_weight)
        if k_weight is not None:
            kw = self._weight(k_weight)
        if inv_freq is not None:
            if inv_freq.dim() != 1 or inv_freq.dtype != self._f32 or not inv_freq.is_contiguous() or inv_freq.device != self.device:
                raise ValueError(f"kv_cache: inv_freq is a float32 vector on {self.device}")
            rot, ip = 2 * inv_freq.shape[0], inv_freq.data_ptr()
        rc = self._append(self._p, layer, tokens, n, cp, sp, heads, qp, qs, k.data_ptr(), ks, v.data_ptr(), vs, op, os_, qw, kw, eps, ip, rot,
                          1 if interleaved else 0, self._raw_stream(index))
        if rc:
            oc.check(rc)
        return q_out

    def _weight(self, w):
        if w.shape != (self.head_dim,) or w.dtype != self.dtype or not w.is_contiguous() or w.device != self.device:
            raise ValueError(f"kv_cache: a norm's weight is [{self.head_dim}] {self.dtype} on {self.device}")
        return w.data_ptr()

    def attention(self, layer, q, cu=None, seqs=None, scale=None, causal=True, window=0, out=None):
        """softmax(scale q . K^T) V of the new tokens' queries [tokens,
        q_heads, head_dim] over their sequences' pages (scale None: 1 /
        sqrt(head_dim)); causal, and the last `window` keys alone when window
        > 0.  `out` may not overlap q.  Rows of `out` behind the last sequence stay as they are (in a new
        tensor: unset); those of an id outside the table are zeros, and check()
        reports it."""
        index = self._index
        if self._current_device() != index:
            with self._torch.cuda.device(index):
                return self.attention(layer, q, cu, seqs, scale, causal, window, out)
        if q.dim() != 3:
            raise ValueError(f"kv_cache: q is [tokens, q_heads, {self.head_dim}], got {tuple(q.shape)}")
        tokens, heads, d = q.shape
        qs = self._rows(q, tokens, heads, "q")
        n, cp, sp = self._batch(tokens, cu, seqs)
        if out is None:
            out = self._empty_like(q)  # contiguous: the heads of q's tokens are
            os_ = heads * d
        else:
            os_ = self._rows(out, tokens, heads, "out")
        need = self._ws_bytes.get((tokens, n, heads)) or self._workspace_size(tokens, n, heads)
        stream = self._raw_stream(index)
        # eager calls of one stream run one after another and share a scratch
        # buffer (of several kernels each, so threads take turns here); a
        # captured call gets its own, which its graph keeps
        with self._turn:
            if self._capturing():
                ws = self._new_bytes(need)
            else:
                ws = self._workspaces.get(stream)
                if ws is None or ws.numel() < need:
                    ws = self._workspaces[stream] = self._new_bytes(need)
            rc = self._attention(self._p, layer, tokens, n, cp, sp, heads, q.data_ptr(), qs, out.data_ptr(), os_,
                                 self._scale if scale is None else scale, 1 if causal else 0, window, ws.data_ptr(), need, stream)
        if rc:
            oc.check(rc)
        return out

    def _workspace_size(self, tokens, n, heads):
        size = oc.sz(0)
        with self._torch.cuda.device(self._index):
            oc.check(oc.lib().oc_kv_attention_workspace_size(self._p, tokens, n, heads, C.byref(size)))
        if len(self._ws_bytes) > 4096:
            self._ws_bytes.clear()
        self._ws_bytes[tokens, n, heads] = need = max(16, size.value)
        return need
