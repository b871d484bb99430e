"""CPU checks of the paged cache's entry points: what the host refuses, before
any device is touched."""
import ctypes as C

import pytest

import kv_cache
import opencuda_cuda as oc


def descriptor(**over):
    """A well-formed cache of made-up addresses (nothing is read on the host)."""
    f = dict(k=0x1000, v=0x2000, page_table=0x3000, seq_len=0x4000, refcount=0x5000, status=0x6000, scratch=0x7000, dtype=2,
             num_layers=2, num_pages=8, kv_heads=4, page_size=16, head_dim=64, max_seqs=4, max_pages_per_seq=4)
    f.update(over)
    return kv_cache._Cache(*(f[name] for name, _ in kv_cache._Cache._fields_))


def size_rc(**over):
    n = C.c_size_t(0)
    return oc.lib().oc_kv_attention_workspace_size(C.byref(descriptor(**over)), 4, 4, 8, C.byref(n))


@pytest.mark.parametrize("over, word", [
    (dict(dtype=3), "dtype"), (dict(k=0), "NULL"), (dict(status=0), "NULL"), (dict(num_layers=0), "empty"), (dict(max_seqs=-1), "empty"),
    (dict(head_dim=257), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(page_size=24), "power of two"), (dict(page_size=2048), "power of two"),
    (dict(k=0x1001), "misaligned"), (dict(max_pages_per_seq=1 << 28), "2^31"), (dict(kv_heads=3), "multiple"),
])
def test_bad_descriptors_are_refused(over, word):
    assert size_rc(**over) == oc.OC_ERR_INVALID_VALUE
    assert word in oc.last_error()


def test_a_good_descriptor_passes():
    assert size_rc() == 0


def attention(c=None, layer=0, tokens=4, n=4, cu=None, heads=8, q=0x100000, qs=512, out=0x200000, os_=512, window=0, ws=0x300000, ws_bytes=0):
    return oc.lib().oc_kv_attention(C.byref(c or descriptor()), layer, tokens, n, cu, None, heads, q, qs, out, os_, 0.125, 1, window, ws, ws_bytes, None)


@pytest.mark.parametrize("args, word", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(n=3), "one token"), (dict(heads=6), "multiple"), (dict(heads=0), "multiple"),
    (dict(q=None), "NULL"), (dict(qs=511), "stride"), (dict(os_=8), "stride"), (dict(window=-1), "window"), (dict(tokens=-1, n=-1), "negative"),
    (dict(ws_bytes=0), "workspace"), (dict(ws=None, ws_bytes=1 << 30), "workspace"), (dict(ws=0x300004, ws_bytes=1 << 30), "workspace"),
    (dict(tokens=1 << 30, n=1 << 30), "too many"),
])
def test_attention_refusals(args, word):
    assert attention(**args) == oc.OC_ERR_INVALID_VALUE
    assert word in oc.last_error()


@pytest.mark.parametrize("args", [
    dict(out=0x100000), dict(out=0x100000 + 2 * 511), dict(out=0x100000 - 2), dict(out=0x100000 + 2 * 512 * 3),
    dict(out=0x100000 + 2 * 512, qs=1023, os_=1023), dict(out=0x100000 + 2 * 600, qs=1024, os_=600), dict(tokens=1, n=1, out=0x100000 + 2),
])
def test_outputs_over_the_queries_are_refused(args):
    assert attention(**args) == oc.OC_ERR_INVALID_VALUE
    assert "overlaps" in oc.last_error()


@pytest.mark.parametrize("args", [
    dict(out=0x100000 + 2 * 512 * 4), dict(out=0x100000 - 2 * 512 * 4), dict(out=0x100000 + 2 * 512, qs=1024, os_=1024),
    dict(out=0x100000 - 2 * 512, qs=1024, os_=1024), dict(out=0x100000 + 2 * 600, qs=1200, os_=1200),
    dict(tokens=1, n=1, out=0x100000 + 2 * 512),
])
def test_outputs_beside_the_queries_pass(args):
    """Other columns of one buffer: the next check is what refuses."""
    assert attention(**args) == oc.OC_ERR_INVALID_VALUE
    assert "workspace" in oc.last_error()


def append(c=None, layer=0, tokens=4, n=4, cu=None, heads=8, q=0x100000, qs=512, k=0x200000, ks=256, v=0x300000, vs=256, qo=0x400000, qos=512,
           inv=None, rot=0):
    return oc.lib().oc_kv_append(C.byref(c or descriptor()), layer, tokens, n, cu, None, heads, q, qs, k, ks, v, vs, qo, qos, None, None, 1e-6, inv,
                                 rot, 0, None)


@pytest.mark.parametrize("args, word", [
    (dict(layer=2), "layer"), (dict(n=3), "one token"), (dict(rot=3, inv=0x9000), "even"), (dict(rot=66, inv=0x9000), "rot_dim"),
    (dict(rot=64), "inv_freq"), (dict(k=None), "NULL"), (dict(qo=None), "NULL"), (dict(ks=255), "stride"), (dict(qs=511), "stride"),
    (dict(tokens=5, n=5), "more entries"), (dict(heads=-1), "negative"), (dict(heads=1 << 26, qs=1 << 33, qos=1 << 33), "too many heads"),
])
def test_append_refusals(args, word):
    assert append(**args) == oc.OC_ERR_INVALID_VALUE
    assert word in oc.last_error()


@pytest.mark.parametrize("args, word", [
    (dict(qo=0x100002), "overlaps q"), (dict(qo=0x100000, qos=1024), "overlaps q"), (dict(qo=0x200000), "overlaps k or v"),
    (dict(qo=0x300000 + 2 * 255), "overlaps k or v"), (dict(qo=0x200000 - 2 * 512, qos=512 + 256, ks=512 + 256, k=0x200000 - 2), "overlaps k or v"),
])
def test_append_over_its_inputs_is_refused(args, word):
    assert append(**args) == oc.OC_ERR_INVALID_VALUE
    assert word in oc.last_error()


def test_empty_batches_do_nothing():
    assert attention(tokens=0, n=0) == 0
    assert append(tokens=0, n=0) == 0
    L, c = oc.lib(), C.byref(descriptor())
    assert L.oc_kv_extend(c, None, None, 0, None) == 0
    assert L.oc_kv_fork(c, None, None, 0, None) == 0
    assert L.oc_kv_free(c, None, 0, None) == 0
    assert L.oc_kv_copy_pages(c, None, None, 0, None) == 0


def test_page_operation_refusals():
    L, c = oc.lib(), C.byref(descriptor())
    for rc in (L.oc_kv_extend(c, None, 0x9000, 1, None), L.oc_kv_extend(c, 0x9000, 0x9000, 5, None), L.oc_kv_fork(c, 0x9000, None, 1, None),
               L.oc_kv_fork(c, 0x9000, 0x9000, 5, None), L.oc_kv_free(c, None, 1, None), L.oc_kv_free(c, 0x9000, -1, None),
               L.oc_kv_copy_pages(c, 0x9000, 0x9000, 9, None), L.oc_kv_copy_pages(c, None, 0x9000, 1, None),
               L.oc_kv_compact(C.byref(descriptor(scratch=0)), None), L.oc_kv_compact(C.byref(descriptor(num_pages=(1 << 20) + 1)), None),
               L.oc_kv_compact(C.byref(descriptor(max_seqs=(1 << 18) + 1)), None), L.oc_kv_compact(None, None)):
        assert rc == oc.OC_ERR_INVALID_VALUE
    n = C.c_size_t(0)
    assert L.oc_kv_scratch_size(0, 4, C.byref(n)) == oc.OC_ERR_INVALID_VALUE
    assert L.oc_kv_scratch_size(8, 4, None) == oc.OC_ERR_INVALID_VALUE
    assert L.oc_kv_scratch_size(8, 4, C.byref(n)) == 0 and n.value >= 4 * (2 * 8 + 4)


def test_python_wrapper_refuses_cpu_tensors():
    import torch
    k = torch.zeros(1, 8, 2, 16, 64)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        kv_cache.KVCache(k, k.clone(), ints(4, 4), ints(4), ints(8))
    with pytest.raises(ValueError):
        kv_cache.KVCache(k.double(), k.double(), ints(4, 4), ints(4), ints(8))
    with pytest.raises(ValueError):
        kv_cache.KVCache(k, k.clone(), ints(4, 4), ints(3), ints(8))
