"""C-ABI checks of the calls around attention that need no GPU: sizes, and arguments refused
before anything is enqueued (a context is opened by the GPU tests only, so device calls are
refused here for their missing context)."""
import ctypes

import pytest

import dyninfer_amd as d

BAD, UNSUPPORTED = d.ERR_INVALID_ARGUMENT, d.ERR_UNSUPPORTED


@pytest.mark.parametrize("kb,k_bits", [(d.KV_Q8, 8), (d.KV_Q4, 4)])
@pytest.mark.parametrize("vb,v_bits", [(d.KV_Q8, 8), (d.KV_Q4, 4)])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("pages,heads,page", [(1, 1, 16), (7, 8, 64), (3, 5, 4096)])
def test_cache_bytes(kb, k_bits, vb, v_bits, dim, pages, heads, page):
    slots = pages * heads * page
    k, v = d.KVCache.bytes(pages, heads, dim, page, kb, vb)
    assert k == slots * (dim * k_bits // 8 + dim // 32 * 2)
    assert v == slots * (dim * v_bits // 8 + 2)


def test_cache_bytes_beyond_32_bits():
    k, _ = d.KVCache.bytes(1 << 20, 8, 128, 256)
    assert k == (1 << 31) * 136


@pytest.mark.parametrize("change,code", [
    (dict(kv_heads=0), BAD), (dict(pages=0), BAD), (dict(kv_heads=5000), UNSUPPORTED), (dict(head_dim=32), UNSUPPORTED),
    (dict(head_dim=112), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED), (dict(page_size=8192), UNSUPPORTED),
    (dict(k_encoding=0), UNSUPPORTED), (dict(v_encoding=9), UNSUPPORTED), (dict(pages=1 << 33), UNSUPPORTED)])
def test_cache_shapes_refused(change, code):
    kw = dict(pages=4, kv_heads=2, head_dim=128, page_size=64)
    kw.update(change)
    with pytest.raises(d.DyninferError) as e:
        d.KVCache.bytes(**kw)
    assert e.value.code == code and e.value.message


def attention_bytes(max_length, max_new=1, tokens=4, seqs=4, heads=32, kv_heads=8, dim=128, dtype=d.DTYPE_BF16):
    cache = d._pack_kvcache(d.KV_Q8, d.KV_Q8, kv_heads, dim, 64, 0, 1, 0, 0, 0, 0)
    batch = d._pack_kvbatch(0, 0, 0, seqs, 1, tokens, max_new, max_length)
    n = ctypes.c_uint64(7)
    rc = d.library().dyninfer_mi355x_tree_attention_workspace_bytes(cache, batch, heads, dtype, ctypes.byref(n))
    return rc, n.value


def test_attention_workspace():
    assert attention_bytes(100) == (0, 0)            # one step: no parts to join
    rc, n = attention_bytes(8192)
    assert rc == 0 and 0 < n < 64 << 20
    assert attention_bytes(8192, seqs=0, tokens=0, max_new=0) == (0, 0)
    assert attention_bytes(8192, seqs=4096) == (0, 0)  # enough units to fill the device whole
    assert attention_bytes(8192, heads=30)[0] == BAD
    assert attention_bytes(8192, heads=0)[0] == BAD
    assert attention_bytes(8192, max_new=5)[0] == BAD  # more rows than tokens
    assert attention_bytes(8192, dtype=d.DTYPE_F16)[0] == UNSUPPORTED
    assert attention_bytes(1 << 40)[0] == UNSUPPORTED
    assert attention_bytes(8192, seqs=1 << 25)[0] == UNSUPPORTED


def test_verify_workspace():
    n = ctypes.c_uint64(0)
    f = d.library().dyninfer_mi355x_draft_verify_workspace_bytes
    assert f(32, 512, 151936, 16, ctypes.byref(n)) == 0 and 0 < n.value < 16 << 20
    assert f(1, 1, 0, 1, ctypes.byref(n)) == BAD
    assert f(1, 1, 10, 2, ctypes.byref(n)) == BAD
    assert f(1, 1, 10, 1, None) == BAD


@pytest.mark.parametrize("name,args", [
    ("rope_table", 5), ("rope", 7), ("kv_append", 9), ("kv_read", 6), ("kv_commit", 7), ("tree_attention", 12),
    ("draft_verify", 5)])
def test_no_context(name, args):
    f = d.library()["dyninfer_mi355x_" + name]  # a fresh handle: plain zero arguments
    f.restype = ctypes.c_int
    types = [ctypes.c_void_p] * args
    if name == "tree_attention":
        types[6] = ctypes.c_float
    f.argtypes = types
    values = [0.0 if t is ctypes.c_float else None for t in types]
    assert f(*values) == BAD
    assert b"context" in d.library().dyninfer_mi355x_last_error()


def test_exported_names_are_listed():
    for name in ("KVCache", "KVBatch", "Rope", "KV_Q8", "KV_Q4"):
        assert name in d.__all__ and hasattr(d, name)
