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


_lib = None


def load_ops_library():
    """Load libcsm_ops.so.  Raises if it is missing -- there is no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(OPS_LIB_PATH):
            raise RuntimeError(f"{OPS_LIB_PATH} not found: build it with `python -m csm_hf_amd.build` (hipcc, gfx950); csm_hf_amd has no CPU fallback")
        lib = C.CDLL(OPS_LIB_PATH)
        for name in OPS_EXPORTS:
            getattr(lib, name).restype = C.c_int
        lib.csm_ops_last_error.restype = C.c_char_p
        if lib.csm_ops_abi_version() != OPS_ABI_VERSION:
            raise RuntimeError(f"libcsm_ops.so ABI {lib.csm_ops_abi_version()} != binding {OPS_ABI_VERSION}")
        lib.csm_ops_paged_rope_append.argtypes = [C.POINTER(RopeAppendArgs), C.c_void_p]
        lib.csm_ops_paged_attention_workspace.argtypes = [C.POINTER(AttentionArgs), C.POINTER(C.c_size_t)]
        lib.csm_ops_paged_prefix_attention.argtypes = [C.POINTER(AttentionArgs), C.c_void_p]
        lib.csm_ops_sample_workspace.argtypes = [C.POINTER(SampleArgs), C.POINTER(C.c_size_t)]
        lib.csm_ops_sample_filtered.argtypes = [C.POINTER(SampleArgs), C.c_void_p]
        _lib = lib
    return _lib


def _ck(lib, rc: int):
    if rc != 0:
        msg = lib.csm_ops_last_error().decode(errors="replace")
        if rc == -3:
            raise ValueError(f"csm_ops capacity error: {msg}")
        raise RuntimeError(f"csm_ops error {rc}: {msg}")


def _call(fn, args, device):
    """One launch on the current stream of `device`."""
    lib = load_ops_library()
    if device.index == torch.cuda.current_device():
        _ck(lib, fn(C.byref(args), torch.cuda.current_stream().cuda_stream))
    else:
        with torch.cuda.device(device):
            _ck(lib, fn(C.byref(args), torch.cuda.current_stream().cuda_stream))


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _on_device(first: torch.Tensor, *named):
    """Every tensor on the GPU of `first`, dense, and none that asks for a gradient."""
    if first.device.type != "cuda":
        raise RuntimeError("csm_hf_amd operators need tensors on the GPU (no CPU fallback)")
    for name, t in named:
        if t is None:
            continue
        if t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, expected {first.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient: this operator has no backward pass (call it under torch.no_grad())")


def _ints(name: str, t: torch.Tensor, shape):
    _need(t.dtype == torch.int32 and tuple(t.shape) == tuple(shape) and t.is_contiguous(), f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}")
    return t.data_ptr()


def _paged(p: PagedArgs, k_cache, v_cache, page_table, seq_lens, cu_rows, rows: int):
    _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype and k_cache.dtype in _DT,
          "k_cache and v_cache must be float32 or bfloat16 tensors [n_pages, n_kv, page_size, head_dim] of one shape and dtype")
    p.n_pages, p.n_kv, p.page_size, p.head_dim = k_cache.shape
    p.k_page_stride, p.k_head_stride, p.k_slot_stride, k_inner = k_cache.stride()
    p.v_page_stride, p.v_head_stride, p.v_slot_stride, v_inner = v_cache.stride()
    _need((k_inner == 1 and v_inner == 1) or p.head_dim == 1, "the last dimension of k_cache and v_cache must be contiguous")
    p.k, p.v, p.dtype = k_cache.data_ptr(), v_cache.data_ptr(), _DT[k_cache.dtype]
    _need(page_table.dim() == 2 and page_table.dtype == torch.int32 and (page_table.shape[1] <= 1 or page_table.stride(1) == 1),
          "page_table must be an int32 tensor [n_seqs, pages] with contiguous rows")
    p.n_seqs, p.table_width = page_table.shape
    p.page_table, p.table_stride = page_table.data_ptr(), page_table.stride(0)
    p.seq_lens = _ints("seq_lens", seq_lens, (p.n_seqs,))
    if cu_rows is not None:
        p.cu_rows = _ints("cu_rows", cu_rows, (p.n_seqs + 1,))
    else:
        _need(rows == p.n_seqs, f"without cu_rows every sequence has one row: {rows} rows, {p.n_seqs} sequences")
    p.rows = rows


def _heads(name: str, t: torch.Tensor, shape, dtype):
    """[rows, heads, dim] with contiguous heads; returns (pointer, row stride)"""
    _need(t.dtype == dtype and tuple(t.shape) == tuple(shape), f"{name} must be a {dtype} tensor of shape {tuple(shape)}")
    _need(t.numel() == 0 or ((t.shape[2] == 1 or t.stride(2) == 1) and (t.shape[1] == 1 or t.stride(1) == t.shape[2])),
          f"the heads of a row of {name} must be contiguous")
    return t.data_ptr(), t.stride(0)


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
    _on_device(qkv, ("qkv", qkv), ("cos", cos), ("sin", sin), ("k_cache", k_cache), ("v_cache", v_cache), ("page_table", page_table),
               ("seq_lens", seq_lens), ("cu_rows", cu_rows), ("q_out", q_out))
    a = RopeAppendArgs()
    _need(qkv.dim() == 2 and qkv.dtype in _DT and (qkv.shape[1] <= 1 or qkv.stride(1) == 1), "qkv must be a float32 or bfloat16 tensor [rows, (n_q + 2 n_kv) * head_dim] with contiguous rows")
    rows = qkv.shape[0]
    _paged(a.c, k_cache, v_cache, page_table, seq_lens, cu_rows, rows)
    hd, n_kv = a.c.head_dim, a.c.n_kv
    n_q = qkv.shape[1] // hd - 2 * n_kv if hd else 0
    _need(n_q >= 1 and qkv.shape[1] == (n_q + 2 * n_kv) * hd, f"qkv rows of {qkv.shape[1]} elements are not n_q + 2 * {n_kv} heads of {hd}")
    for name, t in (("cos", cos), ("sin", sin)):
        _need(t.dtype == torch.float32 and t.dim() == 2 and t.shape[1] == hd // 2 and t.is_contiguous(), f"{name} must be a contiguous float32 tensor [positions, {hd // 2}]")
    _need(cos.shape == sin.shape, "cos and sin must have one shape")
    if q_out is None:
        q_out = torch.empty(rows, n_q, hd, dtype=qkv.dtype, device=qkv.device)
    a.q_out, a.q_out_stride = _heads("q_out", q_out, (rows, n_q, hd), qkv.dtype)
    a.qkv, a.qkv_stride, a.x_dtype, a.n_q = qkv.data_ptr(), qkv.stride(0), _DT[qkv.dtype], n_q
    a.cos, a.sin, a.rope_positions, a.pos_offset = cos.data_ptr(), sin.data_ptr(), cos.shape[0], int(pos_offset)
    _call(load_ops_library().csm_ops_paged_rope_append, a, qkv.device)
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

    A row that sees no key gives zeros.  Rows of padding (`seq_lens < 0`) and rows behind `cu_rows[-1]` keep what `out` held.  Slots on pages
    outside the cache are not seen.  `prefix_len` and all sizes are fixed in a captured graph; lengths, tables and `cu_rows` are read at replay."""
    _on_device(q, ("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("page_table", page_table), ("seq_lens", seq_lens),
               ("prefix_table", prefix_table), ("cu_rows", cu_rows), ("out", out))
    a = AttentionArgs()
    _need(q.dim() == 3 and q.dtype in _DT, "q must be a float32 or bfloat16 tensor [rows, n_q, head_dim]")
    _paged(a.c, k_cache, v_cache, page_table, seq_lens, cu_rows, q.shape[0])
    _need(q.shape[2] == a.c.head_dim, f"q has heads of {q.shape[2]}, the cache of {a.c.head_dim}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    a.q, a.q_stride = _heads("q", q, q.shape, q.dtype)
    a.out, a.out_stride = _heads("out", out, q.shape, q.dtype)
    a.x_dtype, a.n_q = _DT[q.dtype], q.shape[1]
    a.prefix_len = int(prefix_len)
    if prefix_table is not None:
        a.prefix_pages, a.prefix_table = prefix_table.numel(), _ints("prefix_table", prefix_table, (prefix_table.numel(),))
    a.scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    lib = load_ops_library()
    need = C.c_size_t()
    _ck(lib, lib.csm_ops_paged_attention_workspace(C.byref(a), C.byref(need)))
    if need.value:
        ws = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    _call(lib.csm_ops_paged_prefix_attention, a, q.device)
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
    _on_device(logits, ("logits", logits), ("uniform", uniform))
    _need(logits.dim() >= 1 and logits.dtype in _DT, "logits must be a float32 or bfloat16 tensor [..., V]")
    V, lead = logits.shape[-1], logits.shape[:-1]
    lg = logits if logits.dim() == 2 and (V <= 1 or logits.stride(1) == 1) else logits.reshape(-1, V).contiguous()
    rows = lg.shape[0]
    a = SampleArgs()
    keep = []

    def per_row(name, t, dtype):
        _need(t.dtype == dtype and t.numel() == rows and (t.dim() <= 1 or t.shape == lead), f"{name} must be a {dtype} tensor with one value per row")
        if t.device != logits.device:
            raise ValueError(f"{name} is on {t.device}, expected {logits.device}")
        t = t.reshape(-1).contiguous()
        keep.append(t)
        return t.data_ptr()
    a.uniform = per_row("uniform", uniform, torch.float32)
    for name, one, many, value, dtype in (("temperature", "temperature", "temperatures", temperature, torch.float32), ("topk", "topk", "topks", topk, torch.int32),
                                          ("top_p", "top_p", "top_ps", top_p, torch.float32), ("min_p", "min_p", "min_ps", min_p, torch.float32)):
        if torch.is_tensor(value):
            setattr(a, many, per_row(name, value, dtype))
        else:
            setattr(a, one, int(value) if dtype is torch.int32 else float(value))
    out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    a.logits, a.logits_stride, a.x_dtype, a.rows, a.V, a.out = lg.data_ptr(), lg.stride(0), _DT[lg.dtype], rows, V, out.data_ptr()
    lib = load_ops_library()
    need = C.c_size_t()
    _ck(lib, lib.csm_ops_sample_workspace(C.byref(a), C.byref(need)))
    if need.value:
        ws = torch.empty(need.value, dtype=torch.uint8, device=logits.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    _call(lib.csm_ops_sample_filtered, a, logits.device)
    return out.view(*lead, 1)
