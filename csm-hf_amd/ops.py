"""Operators of a serving step over a PAGED KV cache (include/csm_ops.h, libcsm_ops.so), without an engine:

    q = paged_rope_append(qkv, cos, sin, k_cache, v_cache, page_table, seq_lens)      # rotate, append k / v, return rotated q
    o = paged_prefix_attention(q, k_cache, v_cache, page_table, seq_lens, prefix_table=voice_pages, prefix_len=512)
    token = sample_filtered(logits, uniform, temperature=0.9, topk=50, top_p=0.9)

The reference has no paged cache; the arithmetic is that of its decode step (rotary embedding, grouped-query attention and `sample_topk`,
modeling_csm.py:170-189, 345-354), and the tables are `csm_hf_amd.engine.rope_tables`.  All three launch on the CURRENT torch stream of the
tensors' device, do not synchronise, keep nothing between calls and can be captured into a graph.  Inference only: a tensor that asks for a
gradient is refused while gradients are enabled, and so are tensors with a forward-mode tangent and tensors inside a function transform
(`torch.func.vmap`, `jvp`).  There is no CPU fallback."""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional, Union

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
OPS_LIB_PATH = os.path.join(_HERE, "libcsm_ops.so")
OPS_ABI_VERSION = 1
OPS_EXPORTS = ["csm_ops_paged_rope_append", "csm_ops_paged_attention_workspace", "csm_ops_paged_prefix_attention", "csm_ops_sample_workspace",
               "csm_ops_sample_filtered", "csm_ops_last_error", "csm_ops_abi_version"]


# the argument structures of include/csm_ops.h, for callers of the C entries: load_ops_library().csm_ops_sample_filtered(ctypes.byref(args), stream)
class PagedArgs(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int32), ("n_pages", C.c_int32), ("page_size", C.c_int32),
                ("n_kv", C.c_int32), ("head_dim", C.c_int32),
                ("k_page_stride", C.c_int64), ("k_head_stride", C.c_int64), ("k_slot_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_head_stride", C.c_int64), ("v_slot_stride", C.c_int64),
                ("page_table", C.c_void_p), ("table_stride", C.c_int64), ("table_width", C.c_int32), ("n_seqs", C.c_int32),
                ("seq_lens", C.c_void_p), ("cu_rows", C.c_void_p), ("rows", C.c_int32)]


class RopeAppendArgs(C.Structure):
    _fields_ = [("c", PagedArgs), ("qkv", C.c_void_p), ("q_out", C.c_void_p), ("qkv_stride", C.c_int64), ("q_out_stride", C.c_int64),
                ("x_dtype", C.c_int32), ("n_q", C.c_int32), ("cos", C.c_void_p), ("sin", C.c_void_p),
                ("rope_positions", C.c_int32), ("pos_offset", C.c_int32)]


class AttentionArgs(C.Structure):
    _fields_ = [("c", PagedArgs), ("q", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_int64), ("out_stride", C.c_int64),
                ("x_dtype", C.c_int32), ("n_q", C.c_int32), ("prefix_table", C.c_void_p), ("prefix_pages", C.c_int32),
                ("prefix_len", C.c_int32), ("scale", C.c_float), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class SampleArgs(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("logits_stride", C.c_int64), ("x_dtype", C.c_int32), ("rows", C.c_int32), ("V", C.c_int32),
                ("uniform", C.c_void_p), ("temperatures", C.c_void_p), ("top_ps", C.c_void_p), ("min_ps", C.c_void_p), ("topks", C.c_void_p),
                ("temperature", C.c_float), ("top_p", C.c_float), ("min_p", C.c_float), ("topk", C.c_int32), ("out", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


_lib = None
_binding = None


def load_ops_library():
    """Load libcsm_ops.so.  Raises if it is missing -- there is no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(OPS_LIB_PATH):
            raise RuntimeError(f"{OPS_LIB_PATH} not found: build it with `python -m csm_hf_amd.build` (hipcc, gfx950); csm_hf_amd has no CPU fallback")
        lib = C.CDLL(OPS_LIB_PATH)
        for name in OPS_EXPORTS:
            fn = getattr(lib, name)
            fn.restype = C.c_int
            if name.endswith("_workspace"):
                fn.argtypes = [C.c_void_p, C.POINTER(C.c_size_t)]
            elif name not in ("csm_ops_last_error", "csm_ops_abi_version"):
                fn.argtypes = [C.c_void_p, C.c_void_p]
        lib.csm_ops_last_error.restype = C.c_char_p
        if lib.csm_ops_abi_version() != OPS_ABI_VERSION:
            raise RuntimeError(f"libcsm_ops.so ABI {lib.csm_ops_abi_version()} != binding {OPS_ABI_VERSION}")
        _lib = lib
    return _lib


def _load_binding():
    """Load _ops_binding.so (csrc/ops/binding.cpp): the three calls below for torch tensors, checks included."""
    global _binding
    if _binding is None:
        load_ops_library()
        try:
            from . import _ops_binding
        except ImportError as e:
            raise RuntimeError(f"csm_hf_amd/_ops_binding.so is missing or was built against another torch ({e}): build it with `python -m csm_hf_amd.build`") from e
        from .build import binding_stamp
        built_for = getattr(_ops_binding, "built_for", None)   # (None: older than the stamp)
        if built_for != binding_stamp():
            raise RuntimeError(f"csm_hf_amd/_ops_binding.so was built for another torch or Python ({built_for!r}, here: {binding_stamp()!r}): build it with `python -m csm_hf_amd.build`")
        _binding = _ops_binding
    return _binding


def paged_rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      page_table: torch.Tensor, seq_lens: torch.Tensor, *, cu_rows: Optional[torch.Tensor] = None, pos_offset: int = 0,
                      q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of q and k, and k / v written into a paged cache, in one launch; returns the rotated q `[rows, n_q, head_dim]`.

    qkv `[rows, (n_q + 2 n_kv) * head_dim]`: raw q | k | v of each new token row (float32 or bfloat16; rows may be strided).
    cos, sin `[positions, head_dim / 2]` float32 (`engine.rope_tables`); halves rotate like the model's.
    k_cache, v_cache `[n_pages, n_kv, page_size, head_dim]`, float32 or bfloat16, strided views welcome (16-byte strides, page_size a power of two).
    page_table `[n_seqs, pages]` int32: the page of slot s of sequence b is `page_table[b, s // page_size]`.
    seq_lens `[n_seqs]` int32: own slots of each sequence INCLUDING the rows of this call; its row t of T goes to slot `seq_lens - T + t`.
    cu_rows `[n_seqs + 1]` int32: sequence b owns rows `cu_rows[b] : cu_rows[b + 1]`; None = one row per sequence.
    pos_offset: what is added to a slot for its rotary position, i.e. the length of the prefix that precedes the own slots.
    q_out: where the rotated q goes (a new tensor by default); the q part of `qkv` itself is fine.

    A sequence with `seq_lens < 0` is padding.  Its rows, rows behind `cu_rows[-1]` and rows whose slot, page or rotary position lies outside the
    table, the cache or the tables are skipped: nothing is written for them, in q_out either.  Two rows that share a cache slot (a page that
    two sequences write to) leave either row's values there.  q, k and v must not overlap in memory with the cache, nor k_cache with v_cache."""
    return (_binding or _load_binding()).rope_append(qkv, cos, sin, k_cache, v_cache, page_table, seq_lens, cu_rows, pos_offset, q_out)


def paged_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                           prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0, cu_rows: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of new rows over a prefix that the whole batch shares and over each sequence's own slots; `[rows, n_q, head_dim]`.

    q `[rows, n_q, head_dim]` (rotated, unscaled; float32, or bfloat16 over a bfloat16 cache), rows and cache as in `paged_rope_append`, which
    has already appended the rows' own keys.  A row at slot s sees the `prefix_len` slots on the pages `prefix_table` (int32) and own slots 0 .. s.
    The prefix is stored once for the batch, and read once for all rows of a decode batch (sequences with 32 query rows each, and few on a short axis,
    read it with their own slots);
    `prefix_len = 0` is plain paged attention.  `scale` defaults to
    `head_dim ** -0.5`.  head_dim is 64 or 128, n_q any multiple of n_kv.  With float32 q everything is float32; with bfloat16 q the products
    run on the bf16 matrix pipe with float32 sums, the softmax weights of the second one held in 16 bits (two bfloat16 pieces), or rounded to bfloat16
    where the sequences bring more than 16 query rows (`rows * n_q / n_kv`) each on average.

    A row that sees no key gives zeros.  Rows of padding (`seq_lens < 0`) and rows behind `cu_rows[-1]` keep what `out` held (`out` may be `q`).
    Slots on pages outside the cache are not seen.  Slots that no row of the call sees may hold anything; a NaN or infinity in v of a slot that
    some new rows of a sequence see also reaches its earlier rows of the call (0 * NaN), never another sequence.  `prefix_len` and all sizes are fixed in a captured graph; lengths, tables and `cu_rows` are read at replay."""
    return (_binding or _load_binding()).prefix_attention(q, k_cache, v_cache, page_table, seq_lens, prefix_table, prefix_len, cu_rows, scale, out)


def sample_filtered(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Union[float, torch.Tensor] = 1.0,
                    topk: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                    min_p: Union[float, torch.Tensor] = 0.0) -> torch.Tensor:
    """Tokens drawn from `softmax(logits / temperature)` cut by top-k, then top-p, then min-p, with ONE given uniform per row; int32 `[..., 1]`.

    logits `[..., V]` (float32 or bfloat16), uniform `[...]` float32 in [0, 1).  Each setting is a number, or a tensor `[...]` with one value per
    row (float32; int32 for topk).  Numbers are checked: `0 <= temperature < inf`, `0 <= topk <= V`, `0 < top_p <= 1`, `0 <= min_p <= 1`; of a tensor's
    values any is taken, topk <= 0 or >= V, top_p >= 1 and min_p <= 0 as off, others as the nearest that can be used.  Entries are ordered by value, equal ones by index; the kept ones are the first `topk` (0 = all), of these
    the fewest that reach `top_p` of their mass, of these the ones with at least `min_p` times the largest probability; the token is the first
    index at which the running sum of kept probability passes `uniform` times its total.  `temperature = 0` is the arg-max, the lowest index
    of equals, like `sample_topk`; exactly `topk` entries stay, so `topk = 1` is the arg-max too (`sample_topk` keeps every entry that ties with
    the k-th).  V up to 2^21; a NaN logit counts as -inf; a row with nothing but -inf gives -1."""
    return (_binding or _load_binding()).sample(logits, uniform, temperature, topk, top_p, min_p)
