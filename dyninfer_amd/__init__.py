"""dyninfer_amd — MI355X (gfx950) quantized weight-matmul path for dyninfer.

Python host mirror of the C ABI in ``include/dyninfer_mi355x.h`` (the drop-in
boundary).  Every compute call goes through ``libdyninfer_mi355x.so``; there
is no fallback of any kind: if the library is missing or the device is not
gfx950, calls raise.  torch is used only to own device memory and streams.

Reference correspondences:
  * ``QWeight`` — a quantized parameter binding: GGUF ``BlockQuantized`` data
    (crates/dyninfer-checkpoint-gguf/src/convention.rs:200-279) or MLX
    ``GroupQuantized`` packed/scales/biases (crates/dyninfer-checkpoint-safetensors/src/mlx.rs:152-261),
    in their exact on-disk bytes;
  * ``Context.qlinear`` — the helper the selected lowering calls for a
    Linear / OutputProjection (gguf_codegen.rs:268-314, mlx_affine.rs:557-626);
  * ``Context.dequant`` — ``emit_dequant`` (gguf_codegen.rs:350-526);
  * ``candidates`` / ``registry_select`` / ``registry_require`` — kernel
    candidates and ``KernelRegistry::{select,require}``
    (crates/dyninfer-kernel-registry/src/lib.rs:302-399).
"""
from __future__ import annotations

import ctypes
import functools
import json
import os
import struct
from dataclasses import dataclass
from typing import NamedTuple, Optional, Sequence

__all__ = [
    "LIB_PATH", "DyninferError", "QWeight", "Context", "library", "candidates", "registry_select",
    "registry_require", "precision_check", "supports", "ENC_Q4_0", "ENC_Q4_1", "ENC_Q8_0", "ENC_Q6_K", "ENC_Q4_K", "ENC_Q5_K", "ENC_IQ4_XS", "ENC_MLX_U4",
    "DTYPE_F32", "DTYPE_F16", "DTYPE_BF16", "block_geometry", "weight_bytes", "prefill_workspace_bytes",
    "KV_Q8", "KV_Q4", "KVCache", "KVBatch", "Rope", "HeadNorm", "PromptBatch", "TokenLogprobs", "ROPE_INTERLEAVED", "ROPE_HALF", "ROPE_SCALINGS",
    "ERR_INVALID_ARGUMENT",
    "ERR_UNSUPPORTED", "ERR_HIP", "ERR_DEVICE", "ERR_BUFFER_TOO_SMALL",
]

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libdyninfer_mi355x.so")

OK, ERR_INVALID_ARGUMENT, ERR_UNSUPPORTED, ERR_HIP, ERR_DEVICE, ERR_BUFFER_TOO_SMALL = 0, 1, 2, 3, 4, 5
ENC_Q4_0, ENC_Q4_1, ENC_Q8_0, ENC_Q6_K, ENC_MLX_U4 = 2, 3, 8, 14, 0x1004
# GGML's block_q4_K / block_q5_K / block_iq4_xs: schema-only types in the reference (gguf_block.rs:183-316)
ENC_Q4_K, ENC_Q5_K, ENC_IQ4_XS = 12, 13, 23
DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
KV_Q8, KV_Q4 = 1, 2  # DYNINFER_KV_*
ROPE_INTERLEAVED, ROPE_HALF = 0, 1
ROPE_LAYOUTS = {"interleaved": ROPE_INTERLEAVED, "half": ROPE_HALF}
ROPE_SCALINGS = {"none": 0, "linear": 1, "yarn": 2, "bands": 3}
NOALLOC_SCRATCH_BYTES = 32 << 20  # DYNINFER_MI355X_NOALLOC_SCRATCH_BYTES
ENCODING_IDS = {ENC_Q4_0: "gguf.q4_0", ENC_Q4_1: "gguf.q4_1", ENC_Q8_0: "gguf.q8_0", ENC_Q6_K: "gguf.q6_k",
                ENC_Q4_K: "gguf.q4_k", ENC_Q5_K: "gguf.q5_k", ENC_IQ4_XS: "gguf.iq4_xs", ENC_MLX_U4: "mlx.affine.u4"}
# (weights per block, bytes per block): gguf_codegen.rs:23-38; K-quants: gguf_block.rs:207-226
_GGUF_BLOCK = {ENC_Q4_0: (32, 18), ENC_Q4_1: (32, 20), ENC_Q8_0: (32, 34), ENC_Q6_K: (256, 210),
               ENC_Q4_K: (256, 144), ENC_Q5_K: (256, 176), ENC_IQ4_XS: (256, 136)}

EXPORTED_SYMBOLS = (
    "dyninfer_mi355x_open", "dyninfer_mi355x_close", "dyninfer_mi355x_last_error", "dyninfer_mi355x_qlinear",
    "dyninfer_mi355x_qlinear_multi", "dyninfer_mi355x_dequant", "dyninfer_mi355x_embedding", "dyninfer_mi355x_supports",
    "dyninfer_mi355x_gguf_open", "dyninfer_mi355x_gguf_open_memory", "dyninfer_mi355x_gguf_close",
    "dyninfer_mi355x_gguf_tensor_count", "dyninfer_mi355x_gguf_metadata_json", "dyninfer_mi355x_gguf_tensor",
    "dyninfer_mi355x_gguf_find", "dyninfer_mi355x_gguf_upload", "dyninfer_mi355x_gguf_qweight",
    "dyninfer_mi355x_candidates_json", "dyninfer_mi355x_registry_select", "dyninfer_mi355x_registry_require",
    "dyninfer_mi355x_version", "dyninfer_mi355x_qlinear_multi_noalloc", "dyninfer_mi355x_precision_check",
    "dyninfer_mi355x_safetensors_open", "dyninfer_mi355x_safetensors_open_memory", "dyninfer_mi355x_safetensors_close",
    "dyninfer_mi355x_safetensors_tensor_count", "dyninfer_mi355x_safetensors_metadata_json",
    "dyninfer_mi355x_safetensors_tensor", "dyninfer_mi355x_safetensors_find", "dyninfer_mi355x_safetensors_upload",
    "dyninfer_mi355x_safetensors_mlx_qweight", "dyninfer_mi355x_prefill_workspace_bytes",
    "dyninfer_mi355x_rope_table", "dyninfer_mi355x_rope", "dyninfer_mi355x_kv_cache_bytes", "dyninfer_mi355x_kv_append",
    "dyninfer_mi355x_kv_read", "dyninfer_mi355x_kv_commit", "dyninfer_mi355x_tree_attention",
    "dyninfer_mi355x_tree_attention_workspace_bytes", "dyninfer_mi355x_draft_verify",
    "dyninfer_mi355x_draft_verify_workspace_bytes", "dyninfer_mi355x_qk_norm_rope", "dyninfer_mi355x_kv_append_normed",
    "dyninfer_mi355x_prompt_attention", "dyninfer_mi355x_prompt_attention_workspace_bytes",
    "dyninfer_mi355x_token_logprobs", "dyninfer_mi355x_token_logprobs_workspace_bytes",
)


class DyninferError(RuntimeError):
    """Non-zero status from the C ABI; ``code`` is the status, the message is last_error."""

    def __init__(self, code: int, message: str):
        super().__init__(f"[{code}] {message}")
        self.code = code
        self.message = message


class _QWeightC(ctypes.Structure):
    _fields_ = [
        ("encoding", ctypes.c_uint32), ("group_size", ctypes.c_uint32), ("rows", ctypes.c_uint64),
        ("cols", ctypes.c_uint64), ("data", ctypes.c_void_p), ("scales", ctypes.c_void_p),
        ("biases", ctypes.c_void_p), ("scale_dtype", ctypes.c_uint32), ("reserved", ctypes.c_uint32),
        ("data_bytes", ctypes.c_uint64), ("scales_bytes", ctypes.c_uint64), ("biases_bytes", ctypes.c_uint64),
    ]


_pack_qweight = struct.Struct("@2I5Q2I3Q").pack  # _QWeightC's layout

# the descriptors of the calls around attention, as the bytes of their C structs
_pack_kvcache = struct.Struct("@6I5Q").pack
_pack_kvbatch = struct.Struct("@3Q4IQ").pack
_pack_rows = struct.Struct("@Q2I2q").pack
_pack_rope = struct.Struct("@2Q4I").pack
_pack_prompts = struct.Struct("@2Q6I").pack
_pack_head_norm = struct.Struct("@QI2fI").pack
_pack_rope_params = struct.Struct("@2I8d").pack
_pack_logprobs = struct.Struct("@Qq2Q4I5Q").pack
_pack_verify = struct.Struct("@2Q2I2q6Qq4I3Q").pack

_lib: Optional[ctypes.CDLL] = None


class _GgufTensorC(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("type_code", ctypes.c_uint32), ("n_dims", ctypes.c_uint32),
                ("dims", ctypes.c_uint64 * 16), ("offset", ctypes.c_uint64), ("nbytes", ctypes.c_uint64)]


class _StTensorC(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("dtype", ctypes.c_char_p), ("n_dims", ctypes.c_uint32),
                ("dims", ctypes.c_uint64 * 16), ("offset", ctypes.c_uint64), ("nbytes", ctypes.c_uint64)]


def library() -> ctypes.CDLL:
    """Load the built library (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python -m dyninfer_amd.build` "
                          "(the MI355X path has no fallback)")
    lib = ctypes.CDLL(LIB_PATH)
    P, U32, I, SZ = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int, ctypes.c_size_t
    W = ctypes.POINTER(_QWeightC)
    sig = {
        "dyninfer_mi355x_open": (I, [I, ctypes.POINTER(P)]),
        "dyninfer_mi355x_close": (I, [P]),
        "dyninfer_mi355x_last_error": (ctypes.c_char_p, []),
        "dyninfer_mi355x_qlinear": (I, [P, W, P, U32, U32, P, U32, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_qlinear_multi": (I, [P, W, U32, P, U32, U32, ctypes.POINTER(P), U32, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_prefill_workspace_bytes": (I, [W, U32, U32, U32, U32, ctypes.POINTER(ctypes.c_uint64)]),
        "dyninfer_mi355x_qlinear_multi_noalloc": (I, [P, W, U32, P, U32, U32, ctypes.POINTER(P), U32, P]),
        "dyninfer_mi355x_dequant": (I, [P, W, P, P]),
        "dyninfer_mi355x_embedding": (I, [P, W, P, U32, P, P]),
        "dyninfer_mi355x_gguf_open": (I, [ctypes.c_char_p, ctypes.POINTER(P)]),
        "dyninfer_mi355x_gguf_open_memory": (I, [P, ctypes.c_uint64, ctypes.POINTER(P)]),
        "dyninfer_mi355x_gguf_close": (I, [P]),
        "dyninfer_mi355x_gguf_tensor_count": (ctypes.c_uint64, [P]),
        "dyninfer_mi355x_gguf_metadata_json": (ctypes.c_char_p, [P]),
        "dyninfer_mi355x_gguf_tensor": (I, [P, ctypes.c_uint64, ctypes.POINTER(_GgufTensorC)]),
        "dyninfer_mi355x_gguf_find": (I, [P, ctypes.c_char_p, ctypes.POINTER(_GgufTensorC)]),
        "dyninfer_mi355x_gguf_upload": (I, [P, ctypes.c_char_p, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_gguf_qweight": (I, [P, ctypes.c_char_p, P, W]),
        "dyninfer_mi355x_supports": (I, [W, U32, U32, U32]),
        "dyninfer_mi355x_candidates_json": (ctypes.c_char_p, []),
        "dyninfer_mi355x_registry_select": (I, [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_char_p, P, SZ,
                                                ctypes.POINTER(SZ)]),
        "dyninfer_mi355x_registry_require": (I, [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_char_p, P, SZ,
                                                 ctypes.POINTER(SZ)]),
        "dyninfer_mi355x_version": (ctypes.c_char_p, []),
        "dyninfer_mi355x_precision_check": (I, [ctypes.c_char_p, ctypes.c_char_p]),
        "dyninfer_mi355x_safetensors_open": (I, [ctypes.c_char_p, ctypes.POINTER(P)]),
        "dyninfer_mi355x_safetensors_open_memory": (I, [P, ctypes.c_uint64, ctypes.c_char_p, ctypes.POINTER(P)]),
        "dyninfer_mi355x_safetensors_close": (I, [P]),
        "dyninfer_mi355x_safetensors_tensor_count": (ctypes.c_uint64, [P]),
        "dyninfer_mi355x_safetensors_metadata_json": (ctypes.c_char_p, [P]),
        "dyninfer_mi355x_safetensors_tensor": (I, [P, ctypes.c_uint64, ctypes.POINTER(_StTensorC)]),
        "dyninfer_mi355x_safetensors_find": (I, [P, ctypes.c_char_p, ctypes.POINTER(_StTensorC)]),
        "dyninfer_mi355x_safetensors_upload": (I, [P, ctypes.c_char_p, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_safetensors_mlx_qweight": (I, [P, ctypes.c_char_p, P, P, P, W]),
        "dyninfer_mi355x_rope_table": (I, [P, P, U32, P, P]),
        "dyninfer_mi355x_rope": (I, [P, P, P, U32, U32, P, P]),
        "dyninfer_mi355x_kv_cache_bytes": (I, [P, ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_uint64)]),
        "dyninfer_mi355x_kv_append": (I, [P, P, P, P, P, P, P, P, P]),
        "dyninfer_mi355x_qk_norm_rope": (I, [P, P, P, P, P, P, P, U32, U32, P, P]),
        "dyninfer_mi355x_kv_append_normed": (I, [P, P, P, P, P, P, P, P, P, P, P]),
        "dyninfer_mi355x_kv_read": (I, [P, P, P, P, P, P]),
        "dyninfer_mi355x_kv_commit": (I, [P, P, P, P, U32, P, P]),
        "dyninfer_mi355x_tree_attention": (I, [P, P, P, P, P, U32, ctypes.c_float, P, P, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_tree_attention_workspace_bytes": (I, [P, P, U32, U32, ctypes.POINTER(ctypes.c_uint64)]),
        "dyninfer_mi355x_prompt_attention": (I, [P, P, P, P, P, U32, ctypes.c_float, P, P, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_prompt_attention_workspace_bytes": (I, [P, U32, U32, U32, U32, ctypes.POINTER(ctypes.c_uint64)]),
        "dyninfer_mi355x_token_logprobs": (I, [P, P, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_token_logprobs_workspace_bytes": (I, [U32, U32, U32, U32, ctypes.POINTER(ctypes.c_uint64)]),
        "dyninfer_mi355x_draft_verify": (I, [P, P, P, ctypes.c_uint64, P]),
        "dyninfer_mi355x_draft_verify_workspace_bytes": (I, [U32, U32, U32, U32, ctypes.POINTER(ctypes.c_uint64)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    # the calls of every step: the weights as packed bytes (QWeight.pack), see Context
    for name in ("qlinear_multi", "prefill_workspace_bytes", "embedding"):
        fn = lib["dyninfer_mi355x_" + name]
        res, args = sig["dyninfer_mi355x_" + name]
        fn.restype = res
        fn.argtypes = [P if a is W else a for a in args]
        setattr(lib, "packed_" + name, fn)
    _lib = lib
    return lib


def _check(rc: int) -> None:
    if rc != OK:
        raise DyninferError(rc, library().dyninfer_mi355x_last_error().decode())


def block_geometry(encoding: int):
    """(weights per block, bytes per block) of a GGUF encoding."""
    return _GGUF_BLOCK[encoding]


def weight_bytes(encoding: int, rows: int, cols: int, group_size: int = 64, scale_bytes: int = 2) -> int:
    """On-disk weight bytes: the algorithmic HBM traffic of one GEMV pass."""
    if encoding in _GGUF_BLOCK:
        bw, bb = _GGUF_BLOCK[encoding]
        return rows * (cols // bw) * bb
    return rows * cols // 2 + 2 * rows * (cols // group_size) * scale_bytes


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    return t.data_ptr() if hasattr(t, "data_ptr") else int(t)


def _span(t, nbytes: Optional[int]):
    """(address, byte length) of a tensor or raw address; None: a length for the encoding to tell."""
    if t is None:
        return 0, nbytes
    try:
        p = t.data_ptr()
    except AttributeError:
        return int(t), nbytes
    return p, t.numel() * t.element_size() if nbytes is None else nbytes


@dataclass
class QWeight:
    """A quantized weight [rows = N out, cols = K in] in its on-disk bytes.

    GGUF: ``data`` holds the interleaved blocks.  MLX U4: ``data`` = packed u32
    words, ``scales``/``biases`` = [N, K/group] of ``scale_dtype``.  Tensors (or
    raw device addresses) must stay alive while kernels use them.

    Component byte lengths (``*_bytes``) default to the tensors' own sizes, so
    the C ABI checks the buffers actually bound against the encoding's byte
    totals; for a raw address they default to the encoding's expected length.
    """
    encoding: int
    rows: int
    cols: int
    data: object
    scales: object = None
    biases: object = None
    group_size: int = 0
    scale_dtype: int = DTYPE_BF16
    data_bytes: Optional[int] = None
    scales_bytes: Optional[int] = None
    biases_bytes: Optional[int] = None

    def _expected(self):
        if self.encoding in _GGUF_BLOCK:
            bw, bb = _GGUF_BLOCK[self.encoding]
            return self.rows * (self.cols // bw) * bb, 0, 0
        es = 4 if self.scale_dtype == DTYPE_F32 else 2
        g = self.rows * (self.cols // self.group_size) * es if self.group_size else 0
        return self.rows * self.cols // 2, g, g

    def _fields(self):
        """The C struct's values in order."""
        d, dn = _span(self.data, self.data_bytes)
        s, sn = _span(self.scales, self.scales_bytes)
        b, bn = _span(self.biases, self.biases_bytes)
        if dn is None or sn is None or bn is None:
            ed, es, eb = self._expected()
            dn, sn, bn = ed if dn is None else dn, es if sn is None else sn, eb if bn is None else bn
        return (self.encoding, self.group_size, self.rows, self.cols, d, s, b, self.scale_dtype, 0, dn, sn, bn)

    def c(self) -> _QWeightC:
        return _QWeightC(*self._fields())

    def pack(self) -> bytes:
        """The C struct's bytes."""
        v = self._fields()
        try:
            return _pack_qweight(*v)
        except struct.error:  # out of a field's range: wraps as in C, for the library to refuse
            return bytes(_QWeightC(*v))

    @property
    def nbytes(self) -> int:
        sb = 4 if self.scale_dtype == DTYPE_F32 else 2
        return weight_bytes(self.encoding, self.rows, self.cols, self.group_size or 64, sb)


_DTYPE_CODES: dict = {}  # torch dtype -> code, filled on first use (torch is imported late)


def _dtype_code(t) -> int:
    code = _DTYPE_CODES.get(t.dtype)
    if code is not None:
        return code
    import torch
    _DTYPE_CODES.update({torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16})
    if t.dtype not in _DTYPE_CODES:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return _DTYPE_CODES[t.dtype]


def supports(w: QWeight, rows: int, x_dtype: int = DTYPE_F32, y_dtype: int = DTYPE_F32) -> bool:
    wc = w.c()
    return bool(library().dyninfer_mi355x_supports(ctypes.byref(wc), rows, x_dtype, y_dtype))


def prefill_workspace_bytes(ws: Sequence[QWeight], rows: int, x_dtype: int = DTYPE_F32,
                            y_dtype: int = DTYPE_F32) -> int:
    """Device workspace bytes of a qlinear / qlinear_multi call over ``ws`` with these rows
    and dtypes (dyninfer_mi355x_prefill_workspace_bytes): required by a call that runs the
    prefill GEMM, optional for a decode call on the MFMA GEMV (which then stages its
    activations once per call), 0 for every other call."""
    return _workspace_bytes(b"".join([w.pack() for w in ws]), len(ws), rows, x_dtype, y_dtype)


def _workspace_bytes(packed: bytes, count: int, rows: int, x_dtype: int, y_dtype: int) -> int:
    n = ctypes.c_uint64(0)
    rc = library().packed_prefill_workspace_bytes(packed, count, rows, x_dtype, y_dtype, ctypes.byref(n))
    if rc:
        _check(rc)
    return n.value


def _bad(message: str):
    raise DyninferError(ERR_INVALID_ARGUMENT, message)


_T_F32, _T_I32, _T_I64 = 0, 1, 2
_TABLE_DTYPES: list = []  # torch's dtypes of these codes, filled on first use


@functools.lru_cache(maxsize=64)
def _verify_workspace_bytes(seqs: int, tokens: int, vocab: int, max_new: int) -> int:
    """dyninfer_mi355x_draft_verify_workspace_bytes, which depends on these numbers only."""
    need = ctypes.c_uint64(0)
    _check(library().dyninfer_mi355x_draft_verify_workspace_bytes(seqs, tokens, vocab, max_new, ctypes.byref(need)))
    return need.value


@functools.lru_cache(maxsize=64)
def _logprobs_workspace_bytes(rows: int, vocab: int, top: int, dtype: int) -> int:
    """dyninfer_mi355x_token_logprobs_workspace_bytes, which depends on these numbers only."""
    need = ctypes.c_uint64(0)
    _check(library().dyninfer_mi355x_token_logprobs_workspace_bytes(rows, vocab, top, dtype, ctypes.byref(need)))
    return need.value


def _table(t, code: int, shape, what: str) -> int:
    """Address of a contiguous device tensor of that type and shape (None: any length)."""
    if not _TABLE_DTYPES:
        import torch
        _TABLE_DTYPES.extend((torch.float32, torch.int32, torch.int64))
    if t is not None and t.dtype is _TABLE_DTYPES[code] and t.is_cuda and t.is_contiguous():
        s = t.shape
        if s == shape:  # what the callers ask for first, as one comparison
            return t.data_ptr()
        if len(s) == len(shape) and all([n is None or n == m for n, m in zip(shape, s)]):
            return t.data_ptr()
    if t is None:
        _bad(f"{what} is missing")
    want = ", ".join("n" if n is None else str(n) for n in shape)
    _bad(f"{what} must be a contiguous device tensor [{want}] of {('f32', 'int32', 'int64')[code]}")


def _rows(t, tokens: int, dim: int, what: str) -> bytes:
    """The C descriptor of a device tensor [tokens, heads, dim] whose last axis is contiguous."""
    s, st = t.shape, t.stride()
    if not t.is_cuda or len(s) != 3 or s[0] != tokens or s[2] != dim or st[2] != 1:
        _bad(f"{what} must be a device tensor [{tokens}, heads, {dim}] whose last axis is contiguous")
    return _pack_rows(t.data_ptr(), _dtype_code(t), s[1], st[0], st[1])


@dataclass
class KVCache:
    """A paged key/value cache (dyninfer_kvcache_t): uint8 device tensors ``k`` and ``v`` in the
    layout the C header states.  ``KVCache.empty`` allocates them through torch."""
    k: object
    v: object
    pages: int
    kv_heads: int
    head_dim: int
    page_size: int = 64
    k_encoding: int = KV_Q8
    v_encoding: int = KV_Q8

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, k_encoding: int = KV_Q8,
              v_encoding: int = KV_Q8, device="cuda") -> "KVCache":
        import torch
        kb, vb = cls.bytes(pages, kv_heads, head_dim, page_size, k_encoding, v_encoding)
        new = lambda n: torch.empty(n, dtype=torch.uint8, device=device)
        return cls(new(kb), new(vb), pages, kv_heads, head_dim, page_size, k_encoding, v_encoding)

    @staticmethod
    def bytes(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, k_encoding: int = KV_Q8,
              v_encoding: int = KV_Q8):
        """Bytes of the two buffers (dyninfer_mi355x_kv_cache_bytes)."""
        kb, vb = ctypes.c_uint64(0), ctypes.c_uint64(0)
        try:
            packed = _pack_kvcache(k_encoding, v_encoding, kv_heads, head_dim, page_size, 0, pages, 0, 0, 0, 0)
        except struct.error as e:
            _bad(f"cache: {e}")
        _check(library().dyninfer_mi355x_kv_cache_bytes(packed, ctypes.byref(kb), ctypes.byref(vb)))
        return kb.value, vb.value

    def pack(self) -> bytes:
        """The C struct's bytes."""
        k, v = self.k, self.v
        if not (k.is_cuda and v.is_cuda and k.is_contiguous() and v.is_contiguous()):
            _bad("cache buffers must be contiguous device tensors")
        try:
            return _pack_kvcache(self.k_encoding, self.v_encoding, self.kv_heads, self.head_dim, self.page_size, 0,
                                 self.pages, k.data_ptr(), v.data_ptr(), k.nbytes, v.nbytes)
        except struct.error as e:
            _bad(f"cache: {e}")


@dataclass
class KVBatch:
    """The sequences of a call (dyninfer_kvbatch_t): row starts[b] + i of the call's tensors is the
    token at position lengths[b] + i of sequence b.  ``page_table`` [sequences, table_pages],
    ``lengths`` [sequences] and ``starts`` [sequences + 1] are int32 device tensors; ``tokens``
    the rows of the call's tensors, ``max_new`` the most rows of a sequence, ``max_length`` the
    largest length with its rows."""
    page_table: object
    lengths: object
    starts: object
    tokens: int
    max_new: int
    max_length: int

    def pack(self) -> bytes:
        """The C struct's bytes."""
        table, lengths = self.page_table, self.lengths
        n = lengths.shape[0] if lengths.dim() == 1 else -1
        pages = table.shape[1] if table.dim() == 2 else -1
        try:
            return _pack_kvbatch(_table(table, _T_I32, (n, pages), "page_table"), _table(lengths, _T_I32, (n,), "lengths"),
                                 _table(self.starts, _T_I32, (n + 1,), "starts"), n, pages, self.tokens, self.max_new,
                                 self.max_length)
        except struct.error as e:
            _bad(f"batch: {e}")


@dataclass
class Rope:
    """Rotary positions of a call (dyninfer_rope_t): ``table`` [positions, rot_dim / 2, 2] from
    ``Context.rope_table``, ``positions`` int32 [tokens], ``layout`` "interleaved" or "half"."""
    table: object
    positions: object
    rot_dim: int
    layout: str = "half"

    def pack(self, tokens: int) -> bytes:
        """The C struct's bytes."""
        layout = ROPE_LAYOUTS.get(self.layout)
        if layout is None:
            _bad(f"rope layout must be one of {sorted(ROPE_LAYOUTS)}")
        table, rot = self.table, self.rot_dim
        n = table.shape[0] if table.dim() == 3 else -1
        try:
            return _pack_rope(_table(table, _T_F32, (n, rot // 2, 2), "rope table"),
                              _table(self.positions, _T_I32, (tokens,), "positions"), n, rot, layout, 0)
        except struct.error as e:
            _bad(f"rope: {e}")


@dataclass
class PromptBatch:
    """Prompts packed one after the other (dyninfer_prompts_t): rows starts[b] .. starts[b+1] - 1 of
    the queries, int32 [sequences + 1] on the device; ``key_starts`` the same of the keys where
    sequences have more keys than rows (None: as many).  ``max_new`` the most rows of a sequence,
    ``max_keys`` the most keys (without ``key_starts`` those are max_new)."""
    starts: object
    max_new: int
    key_starts: object = None
    max_keys: int = 0

    def pack(self, tokens: int, keys: int) -> bytes:
        """The C struct's bytes."""
        starts, key_starts = self.starts, self.key_starts
        n = starts.shape[0] - 1 if starts.dim() == 1 else -1
        if n < 0:
            _bad("starts must have an element more than there are sequences")
        try:
            return _pack_prompts(_table(starts, _T_I32, (n + 1,), "starts"),
                                 0 if key_starts is None else _table(key_starts, _T_I32, (n + 1,), "key_starts"), n,
                                 tokens, self.max_new, keys, self.max_new if key_starts is None else self.max_keys, 0)
        except struct.error as e:
            _bad(f"batch: {e}")


@dataclass
class HeadNorm:
    """The norm of a head (dyninfer_head_norm_t): x / sqrt(mean(x^2) + eps) * (weight + offset).
    ``weight``: device tensor [head_dim], f32 or bf16, or None (ones)."""
    weight: object = None
    eps: float = 1e-6
    offset: float = 0.0

    def pack(self, dim: int) -> bytes:
        """The C struct's bytes."""
        w = self.weight
        if w is not None and (not w.is_cuda or w.shape != (dim,) or not w.is_contiguous()):
            _bad(f"the norm's weight must be a contiguous device tensor [{dim}]")
        try:
            return _pack_head_norm(0 if w is None else w.data_ptr(), DTYPE_F32 if w is None else _dtype_code(w), self.eps,
                                   self.offset, 0)
        except (struct.error, OverflowError) as e:
            _bad(f"norm: {e}")


class Context:
    """An open library context on one gfx950 device (dyninfer_mi355x_open/close)."""

    def __init__(self, device: int = 0):
        self._lib = library()
        self.device = device
        h = ctypes.c_void_p()
        _check(self._lib.dyninfer_mi355x_open(device, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        """dyninfer_mi355x_close; raises DyninferError on a non-zero status."""
        if getattr(self, "_h", None):
            h, self._h = self._h, None
            _check(self._lib.dyninfer_mi355x_close(h))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # Host time of a call (us; one Q4_0 3072 x 1024 row, three weights of 512 rows, a
    # gather of 512 rows): 12.2, 20.9, 8.2 -> 7.4, 10.8, 5.0.  The C entry takes 3.8, 6.4 and 3.3
    # of it, mostly the launches.  Weights go as packed bytes, built once per call; a
    # caller's workspace goes to the library as it is (it sizes the call itself and
    # leaves a workspace alone that the call has no use for).
    @staticmethod
    def _stream(stream) -> Optional[int]:
        if stream is None:
            import torch
            return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
        return stream if isinstance(stream, int) else stream.cuda_stream

    def _workspace(self, packed: bytes, count: int, x, rows: int, xdt: int, ydt: int, stream, workspace):
        """(pointer, bytes, keep-alive) of the call's device workspace: the caller's
        ``workspace`` tensor, or a new torch allocation of the size the library asks
        for (torch's caching allocator, tied to the launch stream), or none (also when
        ``workspace`` is False: a decode call then runs without its optional one)."""
        if workspace is False:
            return None, 0, None
        if workspace is None:
            need = _workspace_bytes(packed, count, rows, xdt, ydt)
            if need == 0:
                return None, 0, None
            import torch
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
            if stream is not None:
                st = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream))
                workspace.record_stream(st)  # not reused before the call's work on `stream` completes
        return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace

    def qlinear(self, w: QWeight, x, y=None, y_dtype=None, stream=None, workspace=None):
        """y = x · Wᵀ (f32 accumulation).  x: [rows, K] f32 or bf16 device tensor.
        workspace: a device tensor of at least prefill_workspace_bytes([w], rows, …)
        bytes (one is allocated through torch when omitted and that size is not 0), or
        False for none (decode calls only)."""
        return self.qlinear_multi((w,), x, None if y is None else (y,), y_dtype, stream, workspace=workspace)[0]

    def qlinear_multi(self, ws: Sequence[QWeight], x, ys=None, y_dtype=None, stream=None, noalloc=False,
                      workspace=None):
        """One launch for several weights sharing activation x (same encoding and K).
        noalloc: dyninfer_mi355x_qlinear_multi_noalloc (prefill staging in the
        device's static scratch; the caller passes the outputs); otherwise the
        prefill workspace is ``workspace`` or a torch allocation as in qlinear."""
        import torch
        rows = x.shape[0] if x.dim() == 2 else 1
        if ys is None:
            ys = [torch.empty((rows, w.rows), dtype=y_dtype or torch.float32, device=x.device) for w in ws]
        n, xdt, ydt = len(ws), _dtype_code(x), _dtype_code(ys[0])
        yp = (ctypes.c_void_p * n)(*[y.data_ptr() for y in ys])
        if noalloc:
            arr = (_QWeightC * n)(*[w.c() for w in ws])
            _check(self._lib.dyninfer_mi355x_qlinear_multi_noalloc(self._h, arr, n, x.data_ptr(), xdt, rows, yp, ydt,
                                                                   self._stream(stream)))
            return ys
        packed = ws[0].pack() if n == 1 else b"".join([w.pack() for w in ws])
        wp, wn, _keep = self._workspace(packed, n, x, rows, xdt, ydt, stream, workspace)
        _check(self._lib.packed_qlinear_multi(self._h, packed, n, x.data_ptr(), xdt, rows, yp, ydt, wp, wn,
                                              self._stream(stream)))
        return ys

    def dequant(self, w: QWeight, out=None, stream=None):
        """Bit-exact f32 dequantisation of W on the device -> [rows, cols]."""
        import torch
        dev = torch.device("cuda", self.device)
        if out is None:
            out = torch.empty((w.rows, w.cols), dtype=torch.float32, device=dev)
        wc = w.c()
        _check(self._lib.dyninfer_mi355x_dequant(self._h, ctypes.byref(wc), out.data_ptr(), self._stream(stream)))
        return out

    def embedding(self, w: QWeight, ids, out=None, stream=None):
        """Gather rows ids (device int64 [n]) of W and dequantise them -> f32 [n, cols]."""
        import torch
        if ids.dtype != torch.int64 or not ids.is_cuda or not ids.is_contiguous():
            raise DyninferError(ERR_INVALID_ARGUMENT, "ids must be a contiguous int64 device tensor")
        n = ids.numel()
        if out is None:
            out = torch.empty((n, w.cols), dtype=torch.float32, device=ids.device)
        _check(self._lib.packed_embedding(self._h, w.pack(), ids.data_ptr() if n else None, n,
                                         out.data_ptr() if n else None, self._stream(stream)))
        return out

    # ---- around attention: rotary positions, the quantized cache, attention over it, verification
    # Host time of a call (us, small sizes): rope 7.9, kv_append with queries 11.2, kv_read 10.9,
    # kv_commit 7.8, tree_attention 10.6 with one launch and 15.6 with two, draft_verify 20; of it the C entry,
    # mostly its launches, 3.9 a launch, a new output or workspace 1.2 to 1.7, a checked descriptor 0.3 to 1.
    def _on(self, stream) -> int:
        """The raw stream: the given one, or the current one of the context's device."""
        if stream is None:
            import torch
            return torch._C._cuda_getCurrentRawStream(self.device)
        return stream if isinstance(stream, int) else stream.cuda_stream

    @staticmethod
    def _new(shape, dtype, device, stream):
        """A tensor that belongs to the stream the call's work runs on."""
        import torch
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=device)
        st = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream), device=device)
        with torch.cuda.stream(st):
            return torch.empty(shape, dtype=dtype, device=device)

    def _like(self, x, stream):
        """A new tensor of x's shape and type, as _new."""
        if stream is None:
            import torch
            return torch.empty_like(x)
        return self._new(x.shape, x.dtype, x.device, stream)

    def _work(self, need: int, workspace, device, stream):
        """(pointer, bytes, keep-alive) of a call's workspace: the caller's, or a new one."""
        if not need:
            return None, 0, None
        if workspace is None:
            import torch
            workspace = self._new((need,), torch.uint8, device, stream)
        return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace

    def rope_table(self, positions: int, rot_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                   original_length: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                   attn_factor: float = 0.0, low_turns: float = 1.0, high_turns: float = 4.0, out=None, stream=None):
        """Cosines and sines [positions, rot_dim / 2, 2] in f32 (dyninfer_mi355x_rope_table);
        ``scaling``: "none", "linear", "yarn" or "bands"."""
        import torch
        if scaling not in ROPE_SCALINGS:
            _bad(f"rope scaling must be one of {sorted(ROPE_SCALINGS)}")
        if out is None:
            out = self._new((positions, rot_dim // 2, 2), torch.float32, torch.device("cuda", self.device), stream)
        p = _pack_rope_params(rot_dim, ROPE_SCALINGS[scaling], theta, factor, original_length, beta_fast, beta_slow,
                              attn_factor, low_turns, high_turns)
        ptr = _table(out, _T_F32, (positions, rot_dim // 2, 2), "out")
        _check(self._lib.dyninfer_mi355x_rope_table(self._h, p, positions, ptr, self._on(stream)))
        return out

    def rope(self, x, rope: Rope, out=None, stream=None):
        """x [tokens, heads, head_dim] with its first rot_dim dims rotated (dyninfer_mi355x_rope);
        ``out`` may be x."""
        if out is None:
            out = self._like(x, stream)
        n, _, dim = x.shape if x.dim() == 3 else (0, 0, 0)
        _check(self._lib.dyninfer_mi355x_rope(self._h, _rows(x, n, dim, "x"), _rows(out, n, dim, "out"), n, dim,
                                              rope.pack(n), self._on(stream)))
        return out

    def qk_norm_rope(self, q, k=None, rope: Optional[Rope] = None, q_norm: Optional[HeadNorm] = None,
                     k_norm: Optional[HeadNorm] = None, q_out=None, k_out=None, stream=None):
        """q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] with each head by its norm,
        then rotated, in one launch: (q_out, k_out) (dyninfer_mi355x_qk_norm_rope).  Either norm, or
        ``rope``, may be None; q_out may be q, k_out may be k."""
        if q_out is None:
            q_out = self._like(q, stream)
        if k is not None and k_out is None:
            k_out = self._like(k, stream)
        n, _, dim = q.shape if q.dim() == 3 else (0, 0, 0)
        _check(self._lib.dyninfer_mi355x_qk_norm_rope(
            self._h, _rows(q, n, dim, "q"), None if q_norm is None else q_norm.pack(dim), _rows(q_out, n, dim, "q_out"),
            None if k is None else _rows(k, n, dim, "k"), None if k_norm is None else k_norm.pack(dim),
            None if k_out is None else _rows(k_out, n, dim, "k_out"), n, dim, None if rope is None else rope.pack(n),
            self._on(stream)))
        return q_out, k_out

    def kv_append(self, cache: KVCache, batch: KVBatch, k, v, rope: Optional[Rope] = None, q=None, q_out=None,
                  stream=None, q_norm: Optional[HeadNorm] = None, k_norm: Optional[HeadNorm] = None):
        """Quantizes the rows k, v [tokens, kv_heads, head_dim] into the cache, k rotated first if
        ``rope`` is given; then q [tokens, heads, head_dim] is rotated by the same launch and
        returned (dyninfer_mi355x_kv_append).  With ``k_norm`` or ``q_norm`` heads take their norm
        before the rotation (dyninfer_mi355x_kv_append_normed)."""
        n, dim = batch.tokens, cache.head_dim
        if q is not None and q_out is None:
            q_out = self._like(q, stream)
        if q_norm is None and k_norm is None:
            _check(self._lib.dyninfer_mi355x_kv_append(
                self._h, cache.pack(), batch.pack(), _rows(k, n, dim, "k"), _rows(v, n, dim, "v"),
                None if rope is None else rope.pack(n), None if q is None else _rows(q, n, dim, "q"),
                None if q_out is None else _rows(q_out, n, dim, "q_out"), self._on(stream)))
            return q_out
        _check(self._lib.dyninfer_mi355x_kv_append_normed(
            self._h, cache.pack(), batch.pack(), _rows(k, n, dim, "k"), None if k_norm is None else k_norm.pack(dim),
            _rows(v, n, dim, "v"), None if rope is None else rope.pack(n), None if q is None else _rows(q, n, dim, "q"),
            None if q_norm is None else q_norm.pack(dim), None if q_out is None else _rows(q_out, n, dim, "q_out"),
            self._on(stream)))
        return q_out

    def kv_read(self, cache: KVCache, batch: KVBatch, dtype=None, k_out=None, v_out=None, stream=None):
        """The batch's rows of the cache, (k, v) [tokens, kv_heads, head_dim] in ``dtype`` (f32 unless
        given) or into k_out / v_out (dyninfer_mi355x_kv_read)."""
        import torch
        n, dim = batch.tokens, cache.head_dim
        if k_out is None and v_out is None:
            k_out = self._new((n, cache.kv_heads, dim), dtype or torch.float32, cache.k.device, stream)
            v_out = self._like(k_out, stream)
        _check(self._lib.dyninfer_mi355x_kv_read(
            self._h, cache.pack(), batch.pack(), None if k_out is None else _rows(k_out, n, dim, "k_out"),
            None if v_out is None else _rows(v_out, n, dim, "v_out"), self._on(stream)))
        return k_out, v_out

    def kv_commit(self, cache: KVCache, batch: KVBatch, path, counts, stream=None) -> None:
        """Moves the rows of an accepted path (int32 [sequences, width], ``counts`` [sequences], as
        draft_verify returns them) to the front of each sequence's rows (dyninfer_mi355x_kv_commit)."""
        packed = batch.pack()
        n = batch.lengths.shape[0]
        _check(self._lib.dyninfer_mi355x_kv_commit(
            self._h, cache.pack(), packed, _table(path, _T_I32, (n, None), "path"), path.shape[1],
            _table(counts, _T_I32, (n,), "counts"), self._on(stream)))

    def tree_attention(self, cache: KVCache, batch: KVBatch, q, mask=None, scale: Optional[float] = None, out=None,
                       lse=None, stream=None, workspace=None):
        """Attention of q [tokens, heads, head_dim] over the cache, the batch's own rows included
        (dyninfer_mi355x_tree_attention).  ``mask``: int64 [tokens, words], bit j of a row set where it
        sees its sequence's row j; None: a chain.  ``scale``: head_dim ** -0.5 unless given.  ``lse``:
        f32 [tokens, heads] to write the log-sum-exp to."""
        n, dim = batch.tokens, cache.head_dim
        if out is None:
            out = self._like(q, stream)
        qr, cb, bb = _rows(q, n, dim, "q"), cache.pack(), batch.pack()
        mp = None if mask is None else _table(mask, _T_I64, (n, None), "mask")
        if mask is not None and 64 * mask.shape[1] < batch.max_new:
            _bad("mask has fewer bits than max_new")
        lp = None if lse is None else _table(lse, _T_F32, (n, q.shape[1]), "lse")
        need = ctypes.c_uint64(0)
        if workspace is None:
            _check(self._lib.dyninfer_mi355x_tree_attention_workspace_bytes(cb, bb, q.shape[1], _dtype_code(q),
                                                                            ctypes.byref(need)))
            wp, wn, _keep = self._work(need.value, None, q.device, stream)
        else:
            wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        _check(self._lib.dyninfer_mi355x_tree_attention(
            self._h, cb, bb, qr, mp, 0 if mask is None else mask.shape[1], dim ** -0.5 if scale is None else scale,
            _rows(out, n, dim, "out"), lp, wp, wn, self._on(stream)))
        return out

    def tree_attention_workspace_bytes(self, cache: KVCache, batch: KVBatch, q_heads: int, dtype: int = DTYPE_F32) -> int:
        """Device workspace bytes of a tree_attention call (dyninfer_mi355x_tree_attention_workspace_bytes)."""
        need = ctypes.c_uint64(0)
        _check(self._lib.dyninfer_mi355x_tree_attention_workspace_bytes(cache.pack(), batch.pack(), q_heads, dtype,
                                                                        ctypes.byref(need)))
        return need.value

    def prompt_attention(self, q, k, v, batch: PromptBatch, scale: Optional[float] = None, out=None, lse=None, stream=None,
                         workspace=None):
        """Causal attention of q [tokens, heads, head_dim] over k, v [keys, kv_heads, head_dim] of the
        same prompts (dyninfer_mi355x_prompt_attention).  ``scale``: head_dim ** -0.5 unless given.
        ``lse``: f32 [tokens, heads] to write the log-sum-exp to."""
        if out is None:
            out = self._like(q, stream)
        n, heads, dim = q.shape if q.dim() == 3 else (0, 0, 0)
        m, kv_heads = (k.shape[0], k.shape[1]) if k.dim() == 3 else (0, 0)
        qr, kr, vr = _rows(q, n, dim, "q"), _rows(k, m, dim, "k"), _rows(v, m, dim, "v")
        bb = batch.pack(n, m)
        lp = None if lse is None else _table(lse, _T_F32, (n, heads), "lse")
        if workspace is None:
            need = ctypes.c_uint64(0)
            _check(self._lib.dyninfer_mi355x_prompt_attention_workspace_bytes(bb, heads, kv_heads, dim, _dtype_code(q),
                                                                              ctypes.byref(need)))
            wp, wn, _keep = self._work(need.value, None, q.device, stream)
        else:
            wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        _check(self._lib.dyninfer_mi355x_prompt_attention(
            self._h, bb, qr, kr, vr, dim, dim ** -0.5 if scale is None else scale, _rows(out, n, dim, "out"), lp, wp, wn,
            self._on(stream)))
        return out

    def prompt_attention_workspace_bytes(self, batch: PromptBatch, tokens: int, keys: int, q_heads: int, kv_heads: int,
                                         head_dim: int, dtype: int = DTYPE_F32) -> int:
        """Device workspace bytes of a prompt_attention call (dyninfer_mi355x_prompt_attention_workspace_bytes)."""
        need = ctypes.c_uint64(0)
        _check(self._lib.dyninfer_mi355x_prompt_attention_workspace_bytes(batch.pack(tokens, keys), q_heads, kv_heads, head_dim,
                                                                          dtype, ctypes.byref(need)))
        return need.value

    def draft_verify(self, logits, draft_tokens, parents, starts, max_new: int, *, uniform, noise, draft_probs=None,
                     temperature=None, stream=None, workspace=None):
        """Checks drafted trees against the target's logits [tokens, vocab]
        (dyninfer_mi355x_draft_verify): (path int32 [sequences, max_new], counts int32 [sequences],
        next_token int64 [sequences]).  ``parents`` int32 [tokens] or None for chains; ``uniform`` f32
        [tokens], ``noise`` f32 [sequences, vocab] exponentially distributed, ``temperature`` f32
        [sequences] (0: greedy), ``draft_probs`` [tokens, vocab] or None."""
        import torch
        if not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
            _bad("logits must be a device tensor [tokens, vocab] whose last axis is contiguous")
        n, vocab = logits.shape
        seqs = starts.shape[0] - 1 if starts.dim() == 1 else -1
        if draft_probs is not None and (not draft_probs.is_cuda or draft_probs.shape != logits.shape or draft_probs.stride(1) != 1):
            _bad("draft_probs must be a device tensor of the logits' shape whose last axis is contiguous")
        if not noise.is_cuda or noise.dtype != torch.float32 or noise.shape != (seqs, vocab) or noise.stride(1) != 1:
            _bad("noise must be a device tensor [sequences, vocab] of float32 whose last axis is contiguous")
        sp, dp = _table(starts, _T_I32, (None,), "starts"), _table(draft_tokens, _T_I64, (n,), "draft_tokens")
        tp = None if temperature is None else _table(temperature, _T_F32, (seqs,), "temperature")
        pp = None if parents is None else _table(parents, _T_I32, (n,), "parents")
        if stream is None:  # new_empty: 0.3 us less each than torch.empty
            path, counts, token = starts.new_empty((seqs, max_new)), starts.new_empty((seqs,)), draft_tokens.new_empty((seqs,))
        else:
            path = self._new((seqs, max_new), torch.int32, logits.device, stream)
            counts = self._new((seqs,), torch.int32, logits.device, stream)
            token = self._new((seqs,), torch.int64, logits.device, stream)
        wp, wn, _keep = self._work(_verify_workspace_bytes(seqs, n, vocab, max_new), workspace, logits.device, stream)
        args = _pack_verify(
            logits.data_ptr(), 0 if draft_probs is None else draft_probs.data_ptr(), _dtype_code(logits),
            0 if draft_probs is None else _dtype_code(draft_probs), logits.stride(0),
            0 if draft_probs is None else draft_probs.stride(0), dp,
            pp or 0, sp, tp or 0, _table(uniform, _T_F32, (n,), "uniform"), noise.data_ptr(), noise.stride(0),
            vocab, seqs, n, max_new, path.data_ptr(), counts.data_ptr(), token.data_ptr())
        _check(self._lib.dyninfer_mi355x_draft_verify(self._h, args, wp, wn, self._on(stream)))
        return path, counts, token

    def token_logprobs(self, logits, tokens=None, top: int = 0, temperature=None, stream=None, workspace=None):
        """Of logits [rows, vocab]: ``TokenLogprobs`` with the log probabilities of ``tokens`` (int64
        [rows]), their ranks, the entropy, and the ``top`` likeliest tokens with their log probabilities
        (dyninfer_mi355x_token_logprobs).  ``temperature`` f32 [rows] (0: greedy) or None (1).  What is not
        asked for is None."""
        import torch
        if not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
            _bad("logits must be a device tensor [rows, vocab] whose last axis is contiguous")
        n, vocab = logits.shape
        if not isinstance(top, int) or not 0 <= top < 1 << 32:
            _bad("top must be a number of tokens")
        code = _dtype_code(logits)
        kp = 0 if tokens is None else _table(tokens, _T_I64, (n,), "tokens")
        tp = 0 if temperature is None else _table(temperature, _T_F32, (n,), "temperature")
        wp, wn, _keep = self._work(_logprobs_workspace_bytes(n, vocab, top, code), workspace, logits.device, stream)
        logprobs = ranks = top_tokens = top_logprobs = None
        if stream is None:  # new_empty, of the type where a tensor has it: 0.3 to 0.6 us less each than torch.empty
            entropy = logits.new_empty((n,)) if code == DTYPE_F32 else logits.new_empty((n,), dtype=torch.float32)
            if tokens is not None:
                logprobs, ranks = entropy.new_empty((n,)), entropy.new_empty((n,), dtype=torch.int32)
            if top:
                top_logprobs = entropy.new_empty((n, top))
                top_tokens = (entropy if tokens is None else tokens).new_empty((n, top), dtype=torch.int64)
        else:
            new = lambda shape, dtype: self._new(shape, dtype, logits.device, stream)
            entropy = new((n,), torch.float32)
            if tokens is not None:
                logprobs, ranks = new((n,), torch.float32), new((n,), torch.int32)
            if top:
                top_logprobs, top_tokens = new((n, top), torch.float32), new((n, top), torch.int64)
        given = tokens is not None
        args = _pack_logprobs(logits.data_ptr(), logits.stride(0), kp, tp, code, n, vocab, top,
                              logprobs.data_ptr() if given else 0, ranks.data_ptr() if given else 0, entropy.data_ptr(),
                              top_tokens.data_ptr() if top else 0, top_logprobs.data_ptr() if top else 0)
        _check(self._lib.dyninfer_mi355x_token_logprobs(self._h, args, wp, wn, self._on(stream)))
        return TokenLogprobs(logprobs, ranks, entropy, top_tokens, top_logprobs)


class TokenLogprobs(NamedTuple):
    """What ``Context.token_logprobs`` returns."""
    logprobs: object      # f32 [rows], or None without tokens
    ranks: object         # int32 [rows], or None without tokens
    entropy: object       # f32 [rows]
    top_tokens: object    # int64 [rows, top], or None
    top_logprobs: object  # f32 [rows, top], or None


def candidates() -> list:
    """This library's gfx950 KernelCandidateDescriptors (serde JSON)."""
    return json.loads(library().dyninfer_mi355x_candidates_json().decode())


def _registry(fn, request: dict, target: dict, cands) -> dict:
    lib = library()
    cj = None if cands is None else json.dumps(cands).encode()
    rq, tg = json.dumps(request).encode(), json.dumps(target).encode()
    n = ctypes.c_size_t(0)
    rc = getattr(lib, fn)(cj, rq, tg, None, 0, ctypes.byref(n))
    if rc not in (OK, ERR_BUFFER_TOO_SMALL):
        _check(rc)
    buf = ctypes.create_string_buffer(n.value + 1)
    _check(getattr(lib, fn)(cj, rq, tg, ctypes.cast(buf, ctypes.c_void_p), n.value + 1, ctypes.byref(n)))
    return json.loads(buf.value.decode())


def registry_select(request: dict, target: dict, cands=None) -> dict:
    """KernelRegistry::select over ``cands`` (default: this library's candidates) -> SelectionReport."""
    return _registry("dyninfer_mi355x_registry_select", request, target, cands)


def registry_require(request: dict, target: dict, cands=None) -> dict:
    """KernelRegistry::require -> SelectedKernelCandidate, or DyninferError(ERR_UNSUPPORTED, E_KERNEL_COVERAGE…)."""
    return _registry("dyninfer_mi355x_registry_require", request, target, cands)


def precision_check(selected: dict, activation_type: str = "f32") -> None:
    """The compiler's lower.precision gate (crates/dyninfer-compiler/src/lib.rs:289-306),
    relaxed for bf16 activations on this library's lowerings; raises DyninferError
    (ERR_UNSUPPORTED) when the selected kernel is not qualified."""
    _check(library().dyninfer_mi355x_precision_check(json.dumps(selected).encode(), activation_type.encode()))


@dataclass
class GgufTensor:
    name: str
    type_code: int
    shape: tuple
    offset: int
    nbytes: int


class GgufFile:
    """Index of a GGUF file: exact byte ranges of its tensors (dyninfer_mi355x_gguf_*).
    ``GgufFile(path)`` maps the file; ``GgufFile.from_bytes(b)`` indexes bytes in memory."""

    def __init__(self, path: Optional[str] = None, _data=None):
        self._lib = library()
        self._h = ctypes.c_void_p()
        self._keep = None
        if _data is not None:
            self._keep = ctypes.create_string_buffer(bytes(_data), len(_data))
            _check(self._lib.dyninfer_mi355x_gguf_open_memory(ctypes.addressof(self._keep), len(_data),
                                                              ctypes.byref(self._h)))
        else:
            _check(self._lib.dyninfer_mi355x_gguf_open(os.fsencode(path), ctypes.byref(self._h)))

    @classmethod
    def from_bytes(cls, data: bytes) -> "GgufFile":
        return cls(_data=data)

    def close(self) -> None:
        if self._h:
            self._lib.dyninfer_mi355x_gguf_close(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def _py(t: "_GgufTensorC") -> GgufTensor:
        return GgufTensor(t.name.decode(), t.type_code, tuple(t.dims[:t.n_dims]), t.offset, t.nbytes)

    @property
    def tensors(self) -> list:
        out = []
        for i in range(self._lib.dyninfer_mi355x_gguf_tensor_count(self._h)):
            t = _GgufTensorC()
            _check(self._lib.dyninfer_mi355x_gguf_tensor(self._h, i, ctypes.byref(t)))
            out.append(self._py(t))
        return out

    @property
    def metadata(self) -> dict:
        return json.loads(self._lib.dyninfer_mi355x_gguf_metadata_json(self._h).decode())

    def find(self, name: str) -> GgufTensor:
        t = _GgufTensorC()
        _check(self._lib.dyninfer_mi355x_gguf_find(self._h, name.encode(), ctypes.byref(t)))
        return self._py(t)

    def upload(self, name: str, dst=None, stream=None):
        """Copy the tensor's exact bytes to the device (a new uint8 tensor unless dst is given)."""
        import torch
        if dst is None:
            dst = torch.empty(self.find(name).nbytes, dtype=torch.uint8, device="cuda")
        cap = dst.numel() * dst.element_size()
        _check(self._lib.dyninfer_mi355x_gguf_upload(self._h, name.encode(), dst.data_ptr(), cap,
                                                     Context._stream(stream)))
        return dst

    def qweight(self, name: str, device_data) -> QWeight:
        """QWeight of a rank-2 GGUF tensor (Q4_0/Q4_1/Q8_0/Q6_K/Q4_K/Q5_K/IQ4_XS) whose bytes are at device_data."""
        wc = _QWeightC()
        _check(self._lib.dyninfer_mi355x_gguf_qweight(self._h, name.encode(), _ptr(device_data), ctypes.byref(wc)))
        return QWeight(wc.encoding, wc.rows, wc.cols, device_data, data_bytes=wc.data_bytes)


@dataclass
class StTensor:
    name: str
    dtype: str
    shape: tuple
    offset: int
    nbytes: int


class SafeTensorsFile:
    """Index of a .safetensors file (dyninfer_mi355x_safetensors_*): exact byte ranges of its
    tensors and MLX affine weights from their three components.  ``SafeTensorsFile(path)``
    maps the file and reads config.json beside it; ``SafeTensorsFile.from_bytes(b, config)``
    indexes bytes in memory with the text of a config.json (or None)."""

    def __init__(self, path: Optional[str] = None, _data=None, _config: Optional[str] = None):
        self._lib = library()
        self._h = ctypes.c_void_p()
        self._keep = None
        if _data is not None:
            self._keep = ctypes.create_string_buffer(bytes(_data), len(_data))
            cfg = _config.encode() if _config is not None else None
            _check(self._lib.dyninfer_mi355x_safetensors_open_memory(ctypes.addressof(self._keep), len(_data), cfg,
                                                                     ctypes.byref(self._h)))
        else:
            _check(self._lib.dyninfer_mi355x_safetensors_open(os.fsencode(path), ctypes.byref(self._h)))

    @classmethod
    def from_bytes(cls, data: bytes, config: Optional[str] = None) -> "SafeTensorsFile":
        return cls(_data=data, _config=config)

    def close(self) -> None:
        if self._h:
            self._lib.dyninfer_mi355x_safetensors_close(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def _py(t: "_StTensorC") -> StTensor:
        return StTensor(t.name.decode(), t.dtype.decode(), tuple(t.dims[:t.n_dims]), t.offset, t.nbytes)

    @property
    def tensors(self) -> list:
        out = []
        for i in range(self._lib.dyninfer_mi355x_safetensors_tensor_count(self._h)):
            t = _StTensorC()
            _check(self._lib.dyninfer_mi355x_safetensors_tensor(self._h, i, ctypes.byref(t)))
            out.append(self._py(t))
        return out

    @property
    def metadata(self) -> dict:
        return json.loads(self._lib.dyninfer_mi355x_safetensors_metadata_json(self._h).decode())

    def find(self, name: str) -> StTensor:
        t = _StTensorC()
        _check(self._lib.dyninfer_mi355x_safetensors_find(self._h, name.encode(), ctypes.byref(t)))
        return self._py(t)

    def upload(self, name: str, dst=None, stream=None):
        """Copy the tensor's exact bytes to the device (a new uint8 tensor unless dst is given)."""
        import torch
        if dst is None:
            dst = torch.empty(max(self.find(name).nbytes, 1), dtype=torch.uint8, device="cuda")
        cap = dst.numel() * dst.element_size()
        _check(self._lib.dyninfer_mi355x_safetensors_upload(self._h, name.encode(), dst.data_ptr(), cap,
                                                            Context._stream(stream)))
        return dst

    def mlx_qweight(self, weight_name: str, packed, scales, biases) -> QWeight:
        """QWeight of the MLX affine weight `weight_name` whose three components' bytes are at
        packed / scales / biases on the device (validated as the reference's MLX convention)."""
        wc = _QWeightC()
        _check(self._lib.dyninfer_mi355x_safetensors_mlx_qweight(self._h, weight_name.encode(), _ptr(packed),
                                                                 _ptr(scales), _ptr(biases), ctypes.byref(wc)))
        return QWeight(wc.encoding, wc.rows, wc.cols, packed, scales, biases, wc.group_size, wc.scale_dtype,
                       data_bytes=wc.data_bytes, scales_bytes=wc.scales_bytes, biases_bytes=wc.biases_bytes)
