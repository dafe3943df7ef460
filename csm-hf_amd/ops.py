"""Operators of a serving step over a PAGED KV cache (include/csm_ops.h, libcsm_ops.so), without an engine:

    q = paged_rope_append(qkv, cos, sin, k_cache, v_cache, page_table, seq_lens)      # rotate, append k / v, return rotated q
    o = paged_prefix_attention(q, k_cache, v_cache, page_table, seq_lens, prefix_table=voice_pages, prefix_len=512)
    token = sample_filtered(logits, uniform, temperature=0.9, topk=50, top_p=0.9)

The reference has no paged cache; the arithmetic is that of its decode step (rotary embedding, grouped-query attention and `sample_topk`,
modeling_csm.py:170-189, 345-354), and the tables are `csm_hf_amd.engine.rope_tables`.  All three launch on the CURRENT torch stream of the
tensors' device, do not synchronise, keep nothing between calls and can be captured into a graph.  Inference only: a tensor that asks for a
gradient is refused while gradients are enabled.  There is no CPU fallback."""
from __future__ import annotations

import ctypes as C
import os
import struct
from typing import Optional, Union

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
OPS_LIB_PATH = os.path.join(_HERE, "libcsm_ops.so")
OPS_ABI_VERSION = 1
OPS_EXPORTS = ["csm_ops_paged_rope_append", "csm_ops_paged_attention_workspace", "csm_ops_paged_prefix_attention", "csm_ops_sample_workspace",
               "csm_ops_sample_filtered", "csm_ops_last_error", "csm_ops_abi_version"]
_DT = {torch.float32: 0, torch.bfloat16: 1}


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


# A call packs its arguments in one go (setting two dozen ctypes fields takes longer than the smallest kernels run); the ctypes structures above
# describe the same layout.
_P_PAGED = "PPiiiiiqqqqqqPqiiPPi0P"
_PACK_APPEND = struct.Struct("@" + _P_PAGED + "PPqqiiPPii0P").pack
_PACK_ATTENTION = struct.Struct("@" + _P_PAGED + "PPqqiiPiifPN").pack
_PACK_SAMPLE = struct.Struct("@PqiiiPPPPPfffiPPN").pack

_lib = None


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
                fn.argtypes = [C.c_char_p, C.POINTER(C.c_size_t)]
            elif name not in ("csm_ops_last_error", "csm_ops_abi_version"):
                fn.argtypes = [C.c_char_p, C.c_void_p]
        lib.csm_ops_last_error.restype = C.c_char_p
        if lib.csm_ops_abi_version() != OPS_ABI_VERSION:
            raise RuntimeError(f"libcsm_ops.so ABI {lib.csm_ops_abi_version()} != binding {OPS_ABI_VERSION}")
        _lib = lib
    return _lib


def _ck(lib, rc: int):
    msg = lib.csm_ops_last_error().decode(errors="replace")
    if rc == -3:
        raise ValueError(f"csm_ops capacity error: {msg}")
    raise RuntimeError(f"csm_ops error {rc}: {msg}")


_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch.cuda.current_device
_grad_enabled = torch.is_grad_enabled
_int32, _float32 = torch.int32, torch.float32


def _call(fn, args: bytes, device: int):
    """One launch on the current stream of GPU `device`."""
    if device == _current_device():
        rc = fn(args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(args, _raw_stream(device))
    if rc:
        _ck(_lib, rc)


_workspace_sizes = {}


def _workspace(fn, key, args) -> int:
    """Bytes of scratch memory of a call, which depend on the sizes in `key` alone.  The memory itself is allocated by every call."""
    need = _workspace_sizes.get(key)
    if need is None:
        size = C.c_size_t()
        rc = fn(args(), C.byref(size))
        if rc:
            _ck(_lib, rc)
        if len(_workspace_sizes) > 4096:
            _workspace_sizes.clear()
        need = _workspace_sizes[key] = size.value
    return need


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _on_device(named) -> int:
    """The GPU of the first tensor; every other one must be there too, and none may ask for a gradient."""
    dev = named[0][1].get_device()
    if dev < 0:
        raise RuntimeError("csm_hf_amd operators need tensors on the GPU (no CPU fallback)")
    for name, t in named:
        if t is not None:
            if t.get_device() != dev:
                raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
            if t.requires_grad and _grad_enabled():
                raise RuntimeError(f"{name} requires a gradient: this operator has no backward pass (call it under torch.no_grad())")
    return dev


def _index(name: str, v) -> int:
    if type(v) is not int:
        v = int(v)
    if not -0x80000000 <= v <= 0x7fffffff:
        raise ValueError(f"{name} = {v} is out of range")
    return v


def _ints(name: str, t: torch.Tensor, n: int) -> int:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape ({n},)")
    return t.data_ptr()


def _paged(k_cache, v_cache, page_table, seq_lens, cu_rows, rows: int):
    """the fields of csm_ops_paged_t"""
    shape, dtype = k_cache.shape, k_cache.dtype
    dt = _DT.get(dtype)
    if dt is None or len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not dtype:
        raise ValueError("k_cache and v_cache must be float32 or bfloat16 tensors [n_pages, n_kv, page_size, head_dim] of one shape and dtype")
    n_pages, n_kv, page, hd = shape
    strides = k_cache.stride()
    v_strides = strides if k_cache.is_contiguous() and v_cache.is_contiguous() else v_cache.stride()
    if (strides[3] != 1 or v_strides[3] != 1) and hd != 1:
        raise ValueError("the last dimension of k_cache and v_cache must be contiguous")
    if page_table.dim() != 2 or page_table.dtype is not _int32 or not (page_table.is_contiguous() or page_table.stride(1) == 1):
        raise ValueError("page_table must be an int32 tensor [n_seqs, pages] with contiguous rows")
    n_seqs, width = page_table.shape
    if seq_lens.dtype is not _int32 or seq_lens.shape != (n_seqs,) or not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be a contiguous int32 tensor of shape ({n_seqs},)")
    if cu_rows is None:
        cu = 0
        if rows != n_seqs:
            raise ValueError(f"without cu_rows every sequence has one row: {rows} rows, {n_seqs} sequences")
    else:
        cu = _ints("cu_rows", cu_rows, n_seqs + 1)
    return (k_cache.data_ptr(), v_cache.data_ptr(), dt, n_pages, page, n_kv, hd, *strides[:3], *v_strides[:3], page_table.data_ptr(), page_table.stride(0),
            width, n_seqs, seq_lens.data_ptr(), cu, rows)


def _heads(name: str, t: torch.Tensor, shape, dtype):
    """[rows, heads, dim] with contiguous heads; returns (pointer, row stride)"""
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)}")
    if t.is_contiguous():
        return t.data_ptr(), shape[1] * shape[2]
    a, b, c = t.stride()
    if (c != 1 and shape[2] > 1) or (b != shape[2] and shape[1] > 1):
        _need(t.numel() == 0, f"the heads of a row of {name} must be contiguous")
    return t.data_ptr(), a


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
    two sequences write to) leave either row's values there.  q, k and v must not overlap in memory with the cache."""
    dev = _on_device((("qkv", qkv), ("cos", cos), ("sin", sin), ("k_cache", k_cache), ("v_cache", v_cache), ("page_table", page_table),
                           ("seq_lens", seq_lens), ("cu_rows", cu_rows), ("q_out", q_out)))
    x = _DT.get(qkv.dtype)
    if x is None or qkv.dim() != 2 or (qkv.shape[1] > 1 and qkv.stride(1) != 1):
        raise ValueError("qkv must be a float32 or bfloat16 tensor [rows, (n_q + 2 n_kv) * head_dim] with contiguous rows")
    rows, width = qkv.shape
    c = _paged(k_cache, v_cache, page_table, seq_lens, cu_rows, rows)
    n_kv, hd = c[5], c[6]
    n_q = width // hd - 2 * n_kv if hd else 0
    if n_q < 1 or width != (n_q + 2 * n_kv) * hd:
        raise ValueError(f"qkv rows of {width} elements are not n_q + 2 * {n_kv} heads of {hd}")
    half = hd // 2
    positions = cos.shape[0] if cos.dim() else 0
    if cos.dtype is not _float32 or sin.dtype is not _float32 or cos.shape != (positions, half) or sin.shape != (positions, half) or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous float32 tensors [positions, {half}]")
    if q_out is None:
        q_out = qkv.new_empty((rows, n_q, hd))
    q, q_stride = _heads("q_out", q_out, (rows, n_q, hd), qkv.dtype)
    args = _PACK_APPEND(*c, qkv.data_ptr(), q, qkv.stride(0), q_stride, x, n_q, cos.data_ptr(), sin.data_ptr(), positions, _index("pos_offset", pos_offset))
    _call((_lib or load_ops_library()).csm_ops_paged_rope_append, args, dev)
    return q_out


def paged_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                           prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0, cu_rows: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of new rows over a prefix that the whole batch shares and over each sequence's own slots; `[rows, n_q, head_dim]`.

    q `[rows, n_q, head_dim]` (rotated, unscaled; float32, or bfloat16 over a bfloat16 cache), rows and cache as in `paged_rope_append`, which
    has already appended the rows' own keys.  A row at slot s sees the `prefix_len` slots on the pages `prefix_table` (int32) and own slots 0 .. s.
    The prefix is read once for the batch, not once per sequence; `prefix_len = 0` is plain paged attention.  `scale` defaults to
    `head_dim ** -0.5`.  head_dim is 64 or 128, n_q any multiple of n_kv.  With float32 q everything is float32; with bfloat16 q the products
    run on the bf16 matrix pipe with float32 sums and one rounding of the result.

    A row that sees no key gives zeros.  Rows of padding (`seq_lens < 0`) and rows behind `cu_rows[-1]` keep what `out` held (`out` may be `q`).
    Slots on pages outside the cache are not seen.  Slots that no row of the call sees may hold anything; a NaN or infinity in v of a slot that
    some new rows of a sequence see also reaches its earlier rows of the call (0 * NaN), never another sequence.  `prefix_len` and all sizes are fixed in a captured graph; lengths, tables and `cu_rows` are read at replay."""
    dev = _on_device((("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("page_table", page_table), ("seq_lens", seq_lens),
                         ("prefix_table", prefix_table), ("cu_rows", cu_rows), ("out", out)))
    x, shape = _DT.get(q.dtype), q.shape
    if x is None or len(shape) != 3:
        raise ValueError("q must be a float32 or bfloat16 tensor [rows, n_q, head_dim]")
    c = _paged(k_cache, v_cache, page_table, seq_lens, cu_rows, shape[0])
    if shape[2] != c[6]:
        raise ValueError(f"q has heads of {shape[2]}, the cache of {c[6]}")
    if out is None:
        out = q.new_empty(shape)
    pq, q_stride = _heads("q", q, shape, q.dtype)
    po, o_stride = _heads("out", out, shape, q.dtype)
    prefix_len, n_prefix, pp = _index("prefix_len", prefix_len), 0, 0
    if prefix_table is not None:
        n_prefix = prefix_table.numel()
        pp = _ints("prefix_table", prefix_table, n_prefix)
    rest = (pq, po, q_stride, o_stride, x, shape[1], pp, n_prefix, prefix_len, shape[2] ** -0.5 if scale is None else scale)
    lib = _lib or load_ops_library()
    # (what the split of the work goes by: types, sizes of rows, heads, pages and table, prefix)
    need = _workspace(lib.csm_ops_paged_attention_workspace, (shape, x, c[2], c[4], c[5], c[15], c[16], cu_rows is None, prefix_len, n_prefix),
                      lambda: _PACK_ATTENTION(*c, *rest, 0, 0))
    if need:
        ws = q.new_empty(need, dtype=torch.uint8)
        args = _PACK_ATTENTION(*c, *rest, ws.data_ptr(), need)
    else:
        args = _PACK_ATTENTION(*c, *rest, 0, 0)
    _call(lib.csm_ops_paged_prefix_attention, args, dev)
    return out


def sample_filtered(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Union[float, torch.Tensor] = 1.0,
                    topk: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                    min_p: Union[float, torch.Tensor] = 0.0) -> torch.Tensor:
    """Tokens drawn from `softmax(logits / temperature)` cut by top-k, then top-p, then min-p, with ONE given uniform per row; int32 `[..., 1]`.

    logits `[..., V]` (float32 or bfloat16), uniform `[...]` float32 in [0, 1).  Each setting is a number, or a tensor `[...]` with one value per
    row (float32; int32 for topk).  Entries are ordered by value, equal ones by index; the kept ones are the first `topk` (0 = all), of these
    the fewest that reach `top_p` of their mass, of these the ones with at least `min_p` times the largest probability; the token is the first
    index at which the running sum of kept probability passes `uniform` times its total.  `temperature = 0` is the arg-max, the lowest index
    of equals, like `sample_topk`; exactly `topk` entries stay, so `topk = 1` is the arg-max too (`sample_topk` keeps every entry that ties with
    the k-th).  V up to 2^21; a NaN logit counts as -inf; a row with nothing but -inf gives -1."""
    dev = _on_device((("logits", logits), ("uniform", uniform)))
    x, lead = _DT.get(logits.dtype), logits.shape[:-1]
    if x is None or logits.dim() < 1:
        raise ValueError("logits must be a float32 or bfloat16 tensor [..., V]")
    V = logits.shape[-1]
    lg = logits if logits.dim() == 2 and (V <= 1 or logits.stride(1) == 1) else logits.reshape(-1, V).contiguous()
    rows = lg.shape[0]
    keep = []

    def per_row(name, t, dtype):
        if t.dtype is not dtype or t.numel() != rows or (t.dim() > 1 and t.shape != lead):
            raise ValueError(f"{name} must be a {dtype} tensor with one value per row")
        if t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
        if t.dim() != 1 or not t.is_contiguous():
            t = t.reshape(-1).contiguous()
            keep.append(t)
        return t.data_ptr()
    pu = per_row("uniform", uniform, torch.float32)
    one, many = [1.0, 1.0, 0.0, 0], [0, 0, 0, 0]
    for i, (name, value) in enumerate((("temperature", temperature), ("top_p", top_p), ("min_p", min_p), ("topk", topk))):
        if torch.is_tensor(value):
            many[i] = per_row(name, value, torch.int32 if i == 3 else torch.float32)
        else:
            one[i] = _index(name, value) if i == 3 else value
    out = logits.new_empty((*lead, 1), dtype=torch.int32)
    args = (lg.data_ptr(), lg.stride(0), x, rows, V, pu, *many, *one, out.data_ptr())
    lib = _lib or load_ops_library()
    need = _workspace(lib.csm_ops_sample_workspace, (rows, V), lambda: _PACK_SAMPLE(*args, 0, 0)) if V > 4096 else 0
    if need:
        ws = logits.new_empty(need, dtype=torch.uint8)
        packed = _PACK_SAMPLE(*args, ws.data_ptr(), need)
    else:
        packed = _PACK_SAMPLE(*args, 0, 0)
    _call(lib.csm_ops_sample_filtered, packed, dev)
    return out
