"""C-ABI checks, without a GPU, of the calls around prompts: sizes, calls that have nothing to do, and
arguments that are refused before anything is enqueued.  Addresses are numbers that nothing reads: each
call here ends in its checks."""
import ctypes

import pytest

import dyninfer_amd as d

BAD, UNSUPPORTED = d.ERR_INVALID_ARGUMENT, d.ERR_UNSUPPORTED
F32, BF16, F16 = d.DTYPE_F32, d.DTYPE_BF16, d.DTYPE_F16
INF, NAN = float("inf"), float("nan")

# a context's place, for calls that are refused or have nothing to do
CTX = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
A, B, C, D, E, G = (0x10000000 * i for i in range(1, 7))  # far from each other


def message():
    return d.library().dyninfer_mi355x_last_error().decode()


def rows(data=A, dtype=BF16, heads=4, token_stride=None, head_stride=128, dim=128):
    return d._pack_rows(data, dtype, heads, heads * dim if token_stride is None else token_stride, head_stride)


def rope(table=E, positions=E + 0x1000000, count=64, rot=128, layout=d.ROPE_HALF):
    return d._pack_rope(table, positions, count, rot, layout, 0)


def norm(weight=G, dtype=F32, eps=1e-6, offset=0.0):
    return d._pack_head_norm(weight, dtype, eps, offset, 0)


# ---- norms and rotation ----
def qk(q=rows(A), q_norm=norm(), q_out=rows(B), k=rows(C, heads=2), k_norm=norm(), k_out=rows(D, heads=2), tokens=7,
       dim=128, rope=rope()):
    return d.library().dyninfer_mi355x_qk_norm_rope(CTX, q, q_norm, q_out, k, k_norm, k_out, tokens, dim, rope, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dim=32), UNSUPPORTED, "head"), (dict(dim=112), UNSUPPORTED, "head"), (dict(tokens=1 << 31), BAD, "tokens"),
    (dict(k=None), BAD, "together"), (dict(k_out=None), BAD, "together"), (dict(k=None, k_out=None), BAD, "no keys"),
    (dict(rope=None, q_norm=None), BAD, "neither"), (dict(rope=None, k_norm=None), BAD, "neither"),
    (dict(q=None), BAD, "q is NULL"), (dict(q_out=None), BAD, "q_out is NULL"), (dict(q=rows(0)), BAD, "q is NULL"),
    (dict(q=rows(dtype=F16)), UNSUPPORTED, "q must"), (dict(q=rows(A + 1)), BAD, "misaligned"),
    (dict(q=rows(heads=0)), BAD, "no heads"), (dict(q=rows(token_stride=-1)), BAD, "negative"),
    (dict(q_out=rows(B, dtype=F32)), BAD, "share dtype"), (dict(q_out=rows(B, heads=3)), BAD, "share dtype"),
    (dict(k_out=rows(D, heads=4)), BAD, "share dtype"), (dict(k_out=rows(D, dtype=F32, heads=2)), BAD, "share dtype"),
    (dict(q_out=rows(B, token_stride=511)), BAD, "overlap"), (dict(q_out=rows(B, head_stride=127)), BAD, "overlap"),
    (dict(q_out=rows(B, token_stride=0)), BAD, "overlap"),
    (dict(q_out=rows(A + 2)), BAD, "q_out overlaps"), (dict(q_out=rows(A, token_stride=1024)), BAD, "q_out overlaps"),
    (dict(k_out=rows(C + 512, heads=2)), BAD, "k_out overlaps"), (dict(q_out=rows(C)), BAD, "q_out overlaps k"),
    (dict(k_out=rows(A + 256, heads=2)), BAD, "k_out overlaps q"), (dict(k_out=rows(B, heads=2)), BAD, "q_out overlaps k_out"),
    (dict(q_norm=norm(dtype=F16)), UNSUPPORTED, "q_norm"), (dict(k_norm=norm(dtype=F16)), UNSUPPORTED, "k_norm"),
    (dict(q_norm=norm(G + 2)), BAD, "q_norm"), (dict(q_norm=norm(G + 1, BF16)), BAD, "q_norm"),
    (dict(q_norm=norm(eps=0.0)), BAD, "eps"), (dict(q_norm=norm(eps=-1e-6)), BAD, "eps"), (dict(k_norm=norm(eps=NAN)), BAD, "eps"),
    (dict(q_norm=norm(eps=INF)), BAD, "eps"), (dict(q_norm=norm(eps=1e-40)), BAD, "eps"),
    (dict(q_norm=norm(offset=NAN)), BAD, "offset"), (dict(k_norm=norm(offset=INF)), BAD, "offset"),
    (dict(rope=rope(table=0)), BAD, "table"), (dict(rope=rope(table=E + 8)), BAD, "table"),
    (dict(rope=rope(positions=0)), BAD, "positions"), (dict(rope=rope(rot=0)), BAD, "rot_dim"),
    (dict(rope=rope(rot=63)), BAD, "rot_dim"), (dict(rope=rope(rot=130)), BAD, "rot_dim"), (dict(rope=rope(layout=7)), BAD, "layout")])
def test_norms_refused(change, code, text):
    assert qk(**change) == code and text in message()


def test_norms_nothing_to_do():
    assert qk(tokens=0) == 0
    assert qk(tokens=0, q=None, q_out=None) == 0
    assert qk(tokens=0, rope=None) == 0
    assert qk(tokens=0, q_norm=norm(eps=0.0)) == BAD  # still checked


def append(k=rows(A, heads=2), k_norm=norm(), v=rows(B, heads=2), rope=rope(), q=rows(C), q_norm=norm(), q_out=rows(D), tokens=3):
    cache = d._pack_kvcache(d.KV_Q8, d.KV_Q8, 2, 128, 64, 0, 4, 0x70000000, 0x78000000, 4 * 2 * 64 * 136, 4 * 2 * 64 * 130)
    batch = d._pack_kvbatch(0x7C000000, 0x7C100000, 0x7C200000, 3, 4, tokens, min(tokens, 2), 100)
    return d.library().dyninfer_mi355x_kv_append_normed(CTX, cache, batch, k, k_norm, v, rope, q, q_norm, q_out, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(k_norm=norm(eps=0.0)), BAD, "k_norm"), (dict(q_norm=norm(eps=NAN)), BAD, "q_norm"),
    (dict(k_norm=norm(dtype=F16)), UNSUPPORTED, "k_norm"), (dict(k_norm=norm(G + 2)), BAD, "k_norm"),
    (dict(q=None, q_out=None), BAD, "no queries"), (dict(q=None), BAD, "together"), (dict(q_out=None), BAD, "together"),
    (dict(rope=None, q_norm=None), BAD, "no rope"), (dict(k=rows(A, heads=4)), BAD, "heads"),
    (dict(v=rows(B, heads=2, dtype=F32)), BAD, "share a dtype"), (dict(q_out=rows(A)), BAD, "overlaps"),
    (dict(q_out=rows(B + 256)), BAD, "overlaps"), (dict(q_out=rows(C + 256)), BAD, "overlaps"),
    (dict(rope=rope(rot=130)), BAD, "rot_dim")])
def test_normed_append_refused(change, code, text):
    assert append(**change) == code and text in message()


def test_normed_append_nothing_to_do():
    assert append(tokens=0) == 0


# ---- attention of prompts ----
def prompts(starts=E, key_starts=0, seqs=3, tokens=300, max_new=200, keys=300, max_keys=200):
    return d._pack_prompts(starts, key_starts, seqs, tokens, max_new, keys, max_keys, 0)


def attend(batch=prompts(), q=rows(A), k=rows(B, heads=2), v=rows(C, heads=2), dim=128, scale=0.1, out=rows(D), lse=None,
           workspace=None, size=0):
    return d.library().dyninfer_mi355x_prompt_attention(CTX, batch, q, k, v, dim, scale, out, lse, workspace, size, None)


LONG = prompts(key_starts=E + 4096, seqs=1, tokens=4, max_new=4, keys=30000, max_keys=30000)  # split into parts


@pytest.mark.parametrize("change,code,text", [
    (dict(batch=None), BAD, "batch"), (dict(batch=prompts(starts=0)), BAD, "starts"), (dict(batch=prompts(starts=E + 2)), BAD, "starts"),
    (dict(batch=prompts(key_starts=E + 4097)), BAD, "starts"), (dict(batch=prompts(max_new=301)), BAD, "max_new"),
    (dict(batch=prompts(max_keys=301)), BAD, "max_keys"), (dict(batch=prompts(keys=301)), BAD, "key_starts"),
    (dict(batch=prompts(tokens=1 << 31, keys=1 << 31)), BAD, "tokens"),
    (dict(batch=prompts(key_starts=E + 4096, keys=1 << 31)), BAD, "keys"),
    (dict(batch=prompts(seqs=(1 << 24) + 1)), UNSUPPORTED, "sequences"), (dict(dim=48), UNSUPPORTED, "head"),
    (dict(scale=NAN), BAD, "scale"), (dict(scale=-INF), BAD, "scale"), (dict(scale=3e38), BAD, "scale"), (dict(lse=ctypes.c_void_p(G + 2)), BAD, "lse"),
    (dict(q=None), BAD, "q is NULL"), (dict(out=None), BAD, "out is NULL"), (dict(k=None), BAD, "k is NULL"), (dict(v=None), BAD, "v is NULL"),
    (dict(q=rows(A, heads=5), out=rows(D, heads=5)), BAD, "multiple"), (dict(k=rows(B, heads=3), v=rows(C, heads=3)), BAD, "multiple"),
    (dict(v=rows(C, heads=4)), BAD, "share their heads"), (dict(k=rows(B, heads=2, dtype=F32)), BAD, "share a dtype"),
    (dict(q=rows(A, dtype=F16)), UNSUPPORTED, "q must"), (dict(out=rows(D, dtype=F32)), BAD, "share dtype"),
    (dict(out=rows(D, heads=2)), BAD, "share dtype"), (dict(out=rows(D, token_stride=500)), BAD, "overlap"),
    (dict(out=rows(A)), BAD, "overlaps q"), (dict(out=rows(B)), BAD, "overlaps k or v"),
    (dict(out=rows(C + 512)), BAD, "overlaps k or v"), (dict(q=rows(A + 1)), BAD, "misaligned"), (dict(k=rows(B, heads=2, token_stride=-256)), BAD, "negative"),
    (dict(batch=LONG), BAD, "workspace"), (dict(batch=LONG, workspace=ctypes.c_void_p(G), size=16), BAD, "workspace"),
    (dict(batch=LONG, workspace=ctypes.c_void_p(G + 16), size=1 << 30), BAD, "aligned")])
def test_attention_refused(change, code, text):
    assert attend(**change) == code and text in message()


@pytest.mark.parametrize("batch", [
    prompts(seqs=0, starts=0), prompts(tokens=0, max_new=0, keys=0, max_keys=0), prompts(max_new=0),
    prompts(tokens=0, max_new=0, keys=40, max_keys=20, key_starts=E)])
def test_attention_nothing_to_do(batch):
    assert attend(batch=batch) == 0
    assert attend(batch=batch, q=None, k=None, v=None, out=None) == 0


def attention_bytes(seqs, new, prior=0, q_heads=32, kv_heads=8, dim=128, dtype=BF16, out=True):
    t, k = seqs * new, seqs * (new + prior)
    n = ctypes.c_uint64(7)
    rc = d.library().dyninfer_mi355x_prompt_attention_workspace_bytes(
        prompts(0, 1 << 20, seqs, t, new, k, new + prior), q_heads, kv_heads, dim, dtype, ctypes.byref(n) if out else None)
    return rc, n.value


def test_attention_workspace():
    for dtype in (F32, BF16):
        assert attention_bytes(1, 1, dtype=dtype) == (0, 0)
        assert attention_bytes(1, 4096, dtype=dtype) == (0, 0)    # enough rows for the device
        assert attention_bytes(4096, 1, 8191, dtype=dtype) == (0, 0)
        assert attention_bytes(0, 0, dtype=dtype) == (0, 0)
        for dim in (64, 96, 128, 256):
            rc, n = attention_bytes(1, 1, 16000, dim=dim, dtype=dtype)
            assert rc == 0 and 0 < n < 256 << 20 and n % 256 == 0
    assert attention_bytes(1, 1, 2147483646)[0] == 0              # the most keys
    assert attention_bytes(1, 4, q_heads=30)[0] == BAD
    assert attention_bytes(1, 4, kv_heads=0)[0] == BAD
    assert attention_bytes(1, 4, q_heads=0)[0] == BAD
    assert attention_bytes(1, 4, dim=32)[0] == UNSUPPORTED
    assert attention_bytes(1, 4, dtype=F16)[0] == UNSUPPORTED
    assert attention_bytes(1, 4, q_heads=1 << 17, kv_heads=1 << 17)[0] == UNSUPPORTED
    assert attention_bytes(1, 1 << 30, q_heads=32, kv_heads=8)[0] == UNSUPPORTED
    assert attention_bytes(1, 4, out=False)[0] == BAD


# ---- log probabilities ----
def logprobs(logits=A, stride=1000, tokens=B, temperature=0, dtype=BF16, rows=5, vocab=1000, top=3, logprobs=C, ranks=C + 4096,
             entropy=C + 8192, top_tokens=D, top_logprobs=D + 4096, workspace=ctypes.c_void_p(G), size=1 << 30):
    args = d._pack_logprobs(logits, stride, tokens, temperature, dtype, rows, vocab, top, logprobs, ranks, entropy, top_tokens,
                            top_logprobs)
    return d.library().dyninfer_mi355x_token_logprobs(CTX, args, workspace, size, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(vocab=0), BAD, "vocab"), (dict(vocab=1 << 31), BAD, "vocab"), (dict(top=65), UNSUPPORTED, "64 alternatives"),
    (dict(dtype=F16), UNSUPPORTED, "logits"), (dict(logits=0), BAD, "logits"), (dict(logits=A + 1), BAD, "logits"),
    (dict(logits=A + 2, dtype=F32), BAD, "logits"), (dict(stride=999), BAD, "overlap"), (dict(stride=-1000), BAD, "overlap"),
    (dict(tokens=0), BAD, "no tokens"), (dict(tokens=0, ranks=0), BAD, "no tokens"), (dict(tokens=0, logprobs=0), BAD, "no tokens"),
    (dict(tokens=B + 4), BAD, "tokens"), (dict(temperature=B + 2), BAD, "temperature"), (dict(logprobs=C + 2), BAD, "output"),
    (dict(ranks=C + 1), BAD, "output"), (dict(entropy=C + 3), BAD, "output"), (dict(top_tokens=0), BAD, "top_tokens"),
    (dict(top_logprobs=0), BAD, "top_logprobs"), (dict(top_tokens=D + 4), BAD, "top_tokens"), (dict(top_logprobs=D + 2), BAD, "top_logprobs"),
    (dict(vocab=151936, stride=151936, workspace=None), BAD, "workspace"),
    (dict(vocab=151936, stride=151936, size=64), BAD, "workspace"),
    (dict(vocab=151936, stride=151936, workspace=ctypes.c_void_p(G + 8)), BAD, "aligned")])
def test_logprobs_refused(change, code, text):
    assert logprobs(**change) == code and text in message()


def test_logprobs_nothing_to_do():
    assert logprobs(rows=0, logits=0) == 0
    assert d.library().dyninfer_mi355x_token_logprobs(CTX, None, None, 0, None) == BAD


def test_logprobs_workspace():
    def size(rows, vocab, top, dtype=F32, out=True):
        n = ctypes.c_uint64(7)
        rc = d.library().dyninfer_mi355x_token_logprobs_workspace_bytes(rows, vocab, top, dtype, ctypes.byref(n) if out else None)
        return rc, n.value
    for dtype in (F32, BF16):
        rc, n = size(2047, 151936, 5, dtype)
        assert rc == 0 and 0 < n < 64 << 20 and n % 256 == 0
        assert size(8000, 1000, 64, dtype) == (0, 0)   # rows of one piece
        assert size(0, 151936, 5, dtype)[0] == 0
    assert size(1, 0x7FFFFFFF, 64)[0] == 0
    assert size(1, 0, 1)[0] == BAD
    assert size(1, 1 << 31, 1)[0] == BAD
    assert size(1, 10, 65)[0] == UNSUPPORTED
    assert size(1, 10, 1, F16)[0] == UNSUPPORTED
    assert size(1, 10, 1, out=False)[0] == BAD


# ---- all of them ----
@pytest.mark.parametrize("name,args", [
    ("qk_norm_rope", 11), ("kv_append_normed", 11), ("prompt_attention", 12), ("token_logprobs", 5)])
def test_no_context(name, args):
    f = d.library()["dyninfer_mi355x_" + name]  # a fresh handle: plain zero arguments
    f.restype = ctypes.c_int
    types = [ctypes.c_void_p] * args
    if name == "prompt_attention":
        types[6] = ctypes.c_float
    f.argtypes = types
    assert f(*[0.0 if t is ctypes.c_float else None for t in types]) == BAD
    assert "context" in message()


def test_exported_names_are_listed():
    for name in ("HeadNorm", "PromptBatch", "TokenLogprobs"):
        assert name in d.__all__ and hasattr(d, name)
