"""The stand-alone operators of include/csm_ops.h against plain 64-bit implementations: rotary append into a paged cache, attention over a shared
prefix and own pages, filtered sampling -- and the three as one serving step.  Tolerances count roundings (half a step: fp32 2^-24, bf16 2^-8)."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import csm_hf_amd
from csm_hf_amd import ops, paged_rope_append, paged_prefix_attention, sample_filtered

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
DEV = "cuda"


# ---- host side ----------------------------------------------------------------------------------------------------------
def test_library_exports_what_the_header_declares():
    hdr = open(os.path.join(ROOT, "include", "csm_ops.h")).read()
    hdr = re.sub(r"/\*.*?\*/", "", hdr, flags=re.S)
    declared = set(re.findall(r"\b(csm_ops_[a-z0-9_]+)\s*\(", hdr))
    lib = ops.load_ops_library()
    assert declared == set(ops.OPS_EXPORTS) and all(hasattr(lib, n) for n in declared)
    assert lib.csm_ops_abi_version() == ops.OPS_ABI_VERSION
    assert {"paged_rope_append", "paged_prefix_attention", "sample_filtered"} <= set(csm_hf_amd.__all__)


def test_header_is_plain_c_and_structs_match(tmp_path):
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    src = tmp_path / "h.c"
    names = {"csm_ops_paged_t": ops.PagedArgs, "csm_ops_rope_append_t": ops.RopeAppendArgs, "csm_ops_attention_t": ops.AttentionArgs, "csm_ops_sample_t": ops.SampleArgs}
    lines = ["#include <stdio.h>", '#include "csm_ops.h"', "int main(void) {"]
    for n, s in names.items():
        lines.append(f'printf("{n} %zu", sizeof({n}));')
        lines += [f'printf(" %zu", offsetof({n}, {f[0]}));' for f in s._fields_]
        lines.append('printf("\\n");')
    src.write_text("\n".join(lines + ["return 0; }"]))
    r = subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "h")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([str(tmp_path / "h")], capture_output=True, text=True).stdout.split("\n")
    for line, (n, s) in zip(out, names.items()):
        got = line.split()
        assert got == [n, str(C.sizeof(s))] + [str(getattr(s, f[0]).offset) for f in s._fields_]


def _paged_args(p, **over):
    """a valid description of 2 sequences on made-up addresses: only ever handed to calls that must refuse it"""
    for k, v in dict(dict(k=1 << 20, v=1 << 21, dtype=1, n_pages=4, page_size=16, n_kv=2, head_dim=64, k_page_stride=2048, k_head_stride=1024, k_slot_stride=64,
                          v_page_stride=2048, v_head_stride=1024, v_slot_stride=64, page_table=1 << 22, table_stride=2, table_width=2, n_seqs=2,
                          seq_lens=1 << 23, rows=2), **{k: v for k, v in over.items() if hasattr(p, k)}).items():
        setattr(p, k, v)


@pytest.mark.parametrize("over", [
    dict(dtype=2), dict(page_size=24), dict(page_size=0), dict(rows=3), dict(rows=-1), dict(n_kv=0), dict(head_dim=24), dict(head_dim=272), dict(k=(1 << 20) + 8),
    dict(v=None), dict(k_slot_stride=60), dict(v_head_stride=-64), dict(page_table=None), dict(seq_lens=None), dict(x_dtype=3), dict(qkv=None), dict(qkv=(1 << 24) + 2),
    dict(q_out_stride=129), dict(cos=None), dict(q_out_stride=64), dict(k_slot_stride=0), dict(v_page_stride=32), dict(k_head_stride=8), dict(pos_offset=-1), dict(n_q=0), dict(n_q=1 << 29), dict(table_width=1 << 28, page_size=64)])
def test_append_refusals(over):
    lib = ops.load_ops_library()
    a = ops.RopeAppendArgs(qkv=1 << 24, q_out=1 << 25, qkv_stride=384, q_out_stride=128, x_dtype=1, n_q=2, cos=1 << 26, sin=1 << 27, rope_positions=64)
    _paged_args(a.c, **over)
    for k, v in over.items():
        if not hasattr(a.c, k):
            setattr(a, k, v)
    assert lib.csm_ops_paged_rope_append(bytes(a), None) in (-1, -3) and lib.csm_ops_last_error()
    assert lib.csm_ops_paged_rope_append(None, None) == -1


@pytest.mark.parametrize("over", [
    dict(dtype=0), dict(x_dtype=2), dict(head_dim=32), dict(head_dim=96), dict(n_q=3), dict(n_q=0), dict(prefix_len=-1), dict(prefix_len=33, prefix_pages=2, prefix_table=1 << 26),
    dict(prefix_len=5, prefix_pages=1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=(1 << 25) + 4), dict(out_stride=128), dict(out_stride=-256), dict(q_stride=100), dict(rows=1), dict(page_size=3),
    dict(n_pages=(1 << 24) + 1), dict(k_page_stride=1 << 30)])
def test_attention_refusals(over):
    lib = ops.load_ops_library()
    a = ops.AttentionArgs(q=1 << 24, out=1 << 25, q_stride=256, out_stride=256, x_dtype=1, n_q=4, scale=0.125, workspace=1 << 28, workspace_bytes=1 << 27)
    _paged_args(a.c, **over)
    for k, v in over.items():
        if not hasattr(a.c, k):
            setattr(a, k, v)
    need = C.c_size_t()
    assert lib.csm_ops_paged_attention_workspace(bytes(a), C.byref(need)) in (-1, -3)
    assert lib.csm_ops_paged_prefix_attention(bytes(a), None) in (-1, -3) and lib.csm_ops_last_error()


@pytest.mark.parametrize("over", [
    dict(x_dtype=2), dict(rows=-1), dict(V=0), dict(V=(1 << 21) + 1), dict(temperature=-0.5), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(topk=-1), dict(topk=101),
    dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.01), dict(logits=None), dict(uniform=None), dict(out=None)])
def test_sample_refusals(over):
    lib = ops.load_ops_library()
    a = ops.SampleArgs(logits=1 << 20, logits_stride=100, x_dtype=0, rows=2, V=100, uniform=1 << 21, temperature=1.0, top_p=1.0, min_p=0.0, topk=0, out=1 << 22)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.csm_ops_sample_filtered(bytes(a), None) in (-1, -3) and lib.csm_ops_last_error()


def test_small_workspaces_are_refused():
    lib = ops.load_ops_library()
    need = C.c_size_t()
    a = ops.AttentionArgs(q=1 << 24, out=1 << 25, q_stride=256, out_stride=256, x_dtype=1, n_q=4, scale=0.125, prefix_table=1 << 26, prefix_pages=512, prefix_len=8192)
    _paged_args(a.c)
    assert lib.csm_ops_paged_attention_workspace(bytes(a), C.byref(need)) == 0 and need.value > 0
    for ws, size in ((None, 0), (1 << 28, need.value - 1), ((1 << 28) + 4, need.value)):
        a.workspace, a.workspace_bytes = ws, size
        assert lib.csm_ops_paged_prefix_attention(bytes(a), None) == -3
    s = ops.SampleArgs(logits=1 << 20, logits_stride=20000, rows=2, V=20000, uniform=1 << 21, temperature=1.0, top_p=0.5, out=1 << 22)
    assert lib.csm_ops_sample_workspace(bytes(s), C.byref(need)) == 0 and need.value > 0
    for ws, size in ((None, 0), (1 << 28, need.value - 1), ((1 << 28) + 4, need.value)):
        s.workspace, s.workspace_bytes = ws, size
        assert lib.csm_ops_sample_filtered(bytes(s), None) == -3


def test_cpu_tensors_are_refused():
    z, i = torch.zeros(1, 4, 64), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_prefix_attention(z, z[None], z[None], i, i[0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_rope_append(z[0], z[0], z[0], z[None], z[None], i, i[0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sample_filtered(z[0], z[0, :, 0])
    with pytest.raises(TypeError):
        sample_filtered([[1.0]], z)


# ---- plain implementations in 64 bits ------------------------------------------------------------------------------------
class Cache:
    """A paged cache with random contents, scattered pages and lengths; `layout` permutes how pages lie in memory."""

    def __init__(self, lens, page, n_kv, hd, dtype, prefix=0, layout="phsd", seed=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        per = [max(1, -(-max(n, 0) // page)) for n in lens]
        npf = -(-prefix // page)
        n = sum(per) + npf + spare
        order = torch.randperm(n, generator=g).to(torch.int32)
        self.width, self.page, self.n_kv, self.hd, self.prefix_len = max(per) + 1, page, n_kv, hd, prefix
        self.table = torch.full((len(lens), self.width), -7, dtype=torch.int32)
        at = npf
        for b, k in enumerate(per):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.prefix = order[:npf].to(DEV)
        shape = (n, n_kv, page, hd)

        def make(layout):
            perm = {"phsd": (0, 1, 2, 3), "pshd": (0, 2, 1, 3), "hpsd": (1, 0, 2, 3)}[layout]
            x = torch.randn(shape, generator=g).to(dtype)
            y = torch.empty([shape[i] for i in perm], dtype=dtype, device=DEV).permute([perm.index(i) for i in range(4)])
            return y.copy_(x)
        self.k, self.v = (make(l) for l in (("hpsd", "pshd") if layout == "mixed" else (layout, layout)))
        self.table, self.lens = self.table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)

    def args(self):
        return self.k, self.v, self.table, self.lens


def _rows(lens, new):
    """(sequence, slot, row) of every live row"""
    r, out = 0, []
    for b, (n, t) in enumerate(zip(lens, new)):
        out += [(b, n - t + i, r + i) for i in range(t) if n >= 0]
        r += t
    return out, r


def _cu(new):
    return torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def attention64(q, cache, lens, new, n_q, scale, bf16):
    """(result, tolerance) in 64 bits; rows that nothing is written for are NaN.

    Tolerance: a score is a sum of hd products, off by at most (hd + 2) 2^-24 of its absolute sum A in fp32 (2 more for the scale), an exponential
    by that and 2^-21 (the hardware's exp2 and its scaled argument, |argument| < 32); numerator and denominator add n more roundings of 2^-24 each.
    With bf16 operands every probability is one bf16 rounding off at most, and the result one more."""
    rep, hd = n_q // cache.n_kv, cache.hd
    k, v = cache.k.double(), cache.v.double()
    rows, total = _rows(lens, new)
    out = torch.full((total, n_q, hd), math.nan, dtype=torch.float64, device=DEV)
    tol = torch.full_like(out, math.nan)
    flat = lambda z: z.transpose(0, 1).reshape(cache.n_kv, -1, hd)  # noqa: E731
    pk, pv = (flat(z[cache.prefix.long()])[:, :cache.prefix_len] for z in (k, v))
    own = {}
    for b, slot, r in rows:
        if b not in own:
            t = cache.table[b].long()
            own[b] = [flat(z[t[t >= 0]]) for z in (k, v)]
        n = max(0, slot + 1)
        kk, vv = torch.cat((pk, own[b][0][:, :n]), 1), torch.cat((pv, own[b][1][:, :n]), 1)
        qq = q[r].double().view(cache.n_kv, rep, hd)
        if kk.shape[1] == 0:
            out[r], tol[r] = 0.0, 0.0
            continue
        s = qq @ kk.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        o, mag = p @ vv, p @ vv.abs()
        a = (qq.abs() @ kk.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
        rel = 2 * ((hd + 2) * HALF[F32] * a + 2.0 ** -21 + kk.shape[1] * HALF[F32])
        e = mag * (rel + (HALF[BF16] if bf16 else 0.0)) + o.abs() * HALF[BF16 if bf16 else F32]
        out[r], tol[r] = o.reshape(n_q, hd), e.reshape(n_q, hd)
    return out, tol


def check(got, want, tol, untouched):
    """`want` NaN = the row must still hold `untouched`"""
    skip = want.isnan()
    assert bool((got[skip] == untouched).all()), "a row that belongs to nobody was written"
    err = (got.double() - want)[~skip].abs()
    bad = ~(err <= tol[~skip])
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off: worst {float((err / tol[~skip].clamp(min=1e-30)).max())} tolerances, {float(err.max())}"


def sample64(x, u, T, k, p, m):
    x = x.double()
    x = torch.where(x.isnan(), -math.inf, x).tolist()
    mx = max(x)
    if mx == -math.inf:
        return -1
    w = [0.0 if z == -math.inf else 1.0 if z == mx else (0.0 if T == 0 else math.exp((z - mx) / T)) for z in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    k = 1 if T == 0 else len(x) if k <= 0 else k
    order = order[:k]
    if p < 1:
        base, run, n = math.fsum(w[i] for i in order), 0.0, 0
        for n, i in enumerate(order):
            run += w[i]
            if run >= p * base:
                break
        order = order[:n + 1]
    kept = sorted(i for i in order if w[i] >= m or i == order[0])
    total, run = math.fsum(w[i] for i in kept), 0.0
    for i in kept:
        run += w[i]
        if w[i] and run > u * total:
            return i
    return [i for i in kept if w[i]][-1]


# ---- append --------------------------------------------------------------------------------------------------------------
def _append_case(lens, new, n_q, n_kv, hd, x, c, page=16, off=0, layout="phsd", seed=0, in_place=False, wide=0, cu="auto", tail=0):
    cache = Cache(lens, page, n_kv, hd, c, layout=layout, seed=seed)
    live, total = _rows(lens, new)
    g = torch.Generator().manual_seed(seed + 1)
    width = (n_q + 2 * n_kv) * hd
    big = torch.randn(total + tail, width + wide, generator=g).to(x).to(DEV)
    qkv, beside = big[:, :width], big[:, width:].clone()
    src = qkv.clone()
    ang = torch.randn(off + max(max(lens), 1), hd // 2, generator=g, dtype=torch.float64) * 3
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    q_out = qkv[:, :n_q * hd].unflatten(1, (n_q, hd)) if in_place else torch.full((total + tail, n_q, hd), 5.0, dtype=x, device=DEV)
    before = q_out.clone()
    k0, v0 = cache.k.double(), cache.v.double()
    got = paged_rope_append(qkv, cos, sin, *cache.args(), cu_rows=_cu(new) if cu == "auto" else cu, pos_offset=off, q_out=q_out)
    assert got is q_out
    want_q, want_k, want_v = before.double(), k0.clone(), v0.clone()
    tol_q, tol_k = torch.zeros_like(want_q), torch.zeros_like(want_k)
    half = hd // 2
    for b, slot, r in live:
        if slot < 0:
            continue
        h = src[r].double().view(n_q + 2 * n_kv, hd)
        cs, sn = cos[off + slot].double(), sin[off + slot].double()
        lo, hi = h[:n_q + n_kv, :half], h[:n_q + n_kv, half:]
        y = torch.cat((lo * cs - hi * sn, hi * cs + lo * sn), 1)
        e = 2 * HALF[F32] * torch.cat((lo.abs() + hi.abs(),) * 2, 1)      # two products and a sum: at most two fp32 roundings of these terms
        page_no, s = int(cache.table[b, slot // page]), slot % page
        want_q[r], want_k[page_no, :, s], want_v[page_no, :, s] = y[:n_q], y[n_q:], h[n_q + n_kv:]
        tol_q[r] = e[:n_q] + y[:n_q].abs() * HALF[x]
        tol_k[page_no, :, s] = e[n_q:] + y[n_q:].abs() * HALF[c]
    assert bool(((got.double() - want_q).abs() <= tol_q).all())
    assert bool(((cache.k.double() - want_k).abs() <= tol_k).all())
    assert bool(((cache.v.double() - want_v).abs() <= want_v.abs() * HALF[c] * (want_v != v0)).all())
    assert torch.equal(big[:, width:], beside) and torch.equal(qkv[:, n_q * hd:], src[:, n_q * hd:])


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("n_q,n_kv,hd", [(32, 8, 64), (8, 2, 128), (3, 1, 16), (5, 5, 80), (2, 1, 256)])
def test_append_types_and_heads(x, c, n_q, n_kv, hd):
    _append_case([9, 33, 1, 16], [1, 17, 1, 16], n_q, n_kv, hd, x, c, off=5, seed=hd)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 16, 128])
@pytest.mark.parametrize("layout", ["phsd", "pshd", "hpsd", "mixed"])
def test_append_pages_and_layouts(page, layout):
    _append_case([40, 3, 131], [40, 2, 5], 4, 2, 64, BF16, BF16, page=page, layout=layout, wide=64, tail=3)


@pytest.mark.gpu
def test_append_in_place_padding_and_empty_sequences():
    _append_case([4, -1, 7, 0, 2], [2, 3, 0, 0, 2], 4, 2, 64, F32, BF16, in_place=True, tail=2)
    _append_case([4, 1, 7, -1], [1, 1, 1, 1], 4, 2, 64, BF16, BF16, cu=None)          # one row per sequence
    _append_case([1, 5], [3, 2], 4, 2, 64, F32, F32)                                   # more rows than slots: the first two have none
    _append_case([1] * 1500, [i % 2 for i in range(1500)], 2, 1, 64, F32, F32, page=1)  # more sequences than the search keeps on chip


@pytest.mark.gpu
def test_append_skips_what_lies_outside():
    """slots past the table, pages outside the cache, positions past the tables, row offsets that are nonsense: nothing is written"""
    cache = Cache([16, 16, 16, 16], 16, 1, 64, F32)
    cache.table[0, 0], cache.table[1, 0] = cache.k.shape[0], -5
    cache.lens[2] = 16 * cache.width + 1
    qkv = torch.randn(4, 3 * 64, device=DEV)
    tab = torch.zeros(8, 32, device=DEV)
    k0, v0 = cache.k.clone(), cache.v.clone()
    q = torch.full((4, 1, 64), 3.0, device=DEV)
    paged_rope_append(qkv, tab, tab, *cache.args(), q_out=q)                            # sequence 3: slot 15 but only 8 positions
    assert bool((q == 3).all()) and torch.equal(cache.k, k0) and torch.equal(cache.v, v0)
    cache.lens.fill_(2 ** 31 - 1)
    paged_rope_append(qkv, tab, tab, *cache.args(), q_out=q, pos_offset=2 ** 31 - 1)
    cache.lens.fill_(3)
    for cu in ([0, 9, -4, 2 ** 31 - 1, 4], [5, 6, 7, 8, 9], [4, 3, 2, 1, 0], [-2 ** 31, 2 ** 31 - 1, 0, 0, 2]):
        paged_rope_append(qkv, tab, tab, *cache.args(), cu_rows=torch.tensor(cu, dtype=torch.int32, device=DEV), q_out=q)
        torch.cuda.synchronize()
    none = torch.zeros(0, 3 * 64, device=DEV)
    assert paged_rope_append(none, tab, tab, cache.k, cache.v, cache.table[:0], cache.lens[:0]).shape == (0, 1, 64)


# ---- attention -----------------------------------------------------------------------------------------------------------
def _attn_case(lens, new, n_q, n_kv, hd, x, c, page=16, prefix=0, layout="phsd", seed=0, scale=None, gain=1.0, cu="auto", tail=0):
    cache = Cache(lens, page, n_kv, hd, c, prefix=prefix, layout=layout, seed=seed)
    _, total = _rows(lens, new)
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(total + tail, n_q, hd, generator=g) * gain).to(x).to(DEV)
    out = torch.full_like(q, 7.0)
    r = paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix if prefix else None, prefix_len=prefix, cu_rows=_cu(new) if cu == "auto" else cu, scale=scale, out=out)
    assert r is out
    want, tol = attention64(q, cache, lens, new, n_q, hd ** -0.5 if scale is None else scale, x == BF16)
    if tail:
        assert bool((out[total:] == 7).all())
    check(out[:total], want, tol, 7.0)
    return cache, q, out


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("n_q,n_kv,hd", [(32, 8, 64), (8, 2, 128), (1, 1, 64), (6, 6, 128), (14, 2, 64), (40, 1, 128)])
def test_attention_single_tokens(x, c, n_q, n_kv, hd):
    _attn_case([1, 37, 130, -1, 16, 64], [1] * 6, n_q, n_kv, hd, x, c, prefix=45, seed=hd + n_q, cu=None)


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("n_q,n_kv,hd", [(32, 8, 64), (8, 2, 128), (3, 1, 64), (12, 4, 128)])
def test_attention_many_rows(x, c, n_q, n_kv, hd):
    _attn_case([19, 0, 150, -1, 33, 70], [19, 0, 65, 4, 1, 70], n_q, n_kv, hd, x, c, prefix=77, seed=hd + n_q, tail=3)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 1, 15, 64, 333, 2049])
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16)])
def test_attention_prefix_lengths(prefix, x, c):
    _attn_case([5, 600, 1], [1, 1, 1], 8, 2, 64, x, c, prefix=prefix, seed=prefix)
    _attn_case([5, 40, 100], [5, 3, 100], 8, 2, 64, x, c, prefix=prefix, seed=prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 4, 32, 128, 1024])
@pytest.mark.parametrize("layout", ["phsd", "pshd", "hpsd", "mixed"])
def test_attention_pages_and_layouts(page, layout):
    _attn_case([3, 77, 200], [1, 1, 1], 4, 2, 64, BF16, BF16, page=page, prefix=50, layout=layout)
    _attn_case([30, 77], [30, 50], 4, 2, 128, F32, BF16, page=page, prefix=21, layout=layout)
    _attn_case([30, 77], [30, 50], 4, 2, 64, BF16, BF16, page=page, prefix=21, layout=layout)
    _attn_case([30, 77], [1, 50], 4, 2, 64, F32, F32, page=page, prefix=21, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("b,longest,prefix", [(1, 1, 0), (1, 2048, 0), (2, 5000, 0), (130, 40, 100), (300, 3, 17), (1, 1, 8192), (64, 1, 1)])
@pytest.mark.parametrize("x", [BF16, F32])
def test_attention_sizes(b, longest, prefix, x):
    lens = [max(1, longest - (i * 37) % (longest // 2 + 1)) for i in range(b)]
    _attn_case(lens, [1] * b, 8, 2, 64, x, BF16, prefix=prefix, page=32, seed=b, cu=None)


@pytest.mark.gpu
@pytest.mark.parametrize("x", [BF16, F32])
def test_attention_sharp_scores_and_other_scales(x):
    """scores of hundreds (a softmax that is one key), a scale of 0 (a plain mean) and a negative scale"""
    _attn_case([90, 300], [1, 40], 4, 2, 64, x, BF16, prefix=70, gain=30.0)
    _attn_case([90, 300], [1, 40], 4, 2, 64, x, BF16, prefix=70, scale=0.0)
    _attn_case([90, 300], [1, 40], 4, 2, 64, x, BF16, prefix=70, scale=-0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("x", [BF16, F32])
def test_attention_rows_without_keys(x):
    """no prefix and a length of zero, or more rows than slots: rows that see nothing are zero"""
    _attn_case([0, 2, 5], [0, 4, 5], 4, 2, 64, x, BF16)
    _attn_case([0, 0, 3], [1, 1, 1], 4, 2, 64, x, BF16, cu=None)
    cache = Cache([0], 16, 1, 64, BF16)
    q = torch.randn(1, 2, 64, device=DEV).to(x)
    cache.table = cache.table[:, :0]                                   # a table without a page
    assert bool((paged_prefix_attention(q, *cache.args()) == 0).all())
    assert paged_prefix_attention(q[:0], cache.k, cache.v, cache.table[:0], cache.lens[:0]).shape == (0, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("x", [BF16, F32])
@pytest.mark.parametrize("new", [[1, 1], [20, 20]])
def test_attention_never_reads_what_is_not_seen(x, new):
    """NaN and infinity in every slot past the lengths, on unused pages and on pages of other sequences change nothing; pages outside the cache hide their slots"""
    lens, prefix = [21, 20], 19
    cache = Cache(lens, 16, 2, 64, BF16, prefix=prefix)
    seen = torch.zeros(cache.k.shape[0], 16, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for s in range(n):
            seen[cache.table[b, s // 16], s % 16] = True
    for s in range(prefix):
        seen[cache.prefix[s // 16], s % 16] = True
    q = torch.randn(sum(new), 4, 64, device=DEV).to(x)
    run = lambda: paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=prefix, cu_rows=_cu(new))  # noqa: E731
    want, tol = attention64(q, cache, lens, new, 4, 0.125, x == BF16)
    hidden = (~seen)[:, None, :, None].expand_as(cache.k)
    for junk in (math.nan, math.inf, -math.inf, 3e38):
        cache.k[hidden], cache.v[hidden] = junk, junk
        check(run(), want, tol, 0.0)
    page = int(cache.table[0, 0])
    for bad in (-1, cache.k.shape[0], 2 ** 31 - 1, -2 ** 31):        # sequence 0 loses its first page
        cache.table[0, 0] = bad
        got = run()
        kk = torch.cat([cache.k[cache.prefix.long()].transpose(0, 1).reshape(2, -1, 64)[:, :prefix], cache.k[cache.table[0, 1].long()][:, :5]], 1).double()
        vv = torch.cat([cache.v[cache.prefix.long()].transpose(0, 1).reshape(2, -1, 64)[:, :prefix], cache.v[cache.table[0, 1].long()][:, :5]], 1).double()
        last = new[0] - 1
        p = torch.softmax(q[last].double().view(2, 2, 64) @ kk.transpose(1, 2) * 0.125, -1)
        assert float(((p @ vv).view(4, 64) - got[last].double()).abs().max()) < (2.0 ** -6 if x == BF16 else 1e-4)
        check(got[new[0]:], want[new[0]:], tol[new[0]:], 0.0)
    cache.table[0, 0] = page
    cache.prefix = cache.prefix.clone()
    keep = int(cache.prefix[1])
    cache.prefix[1] = -3
    a = run()
    cache.prefix[1] = keep
    b = paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=16, cu_rows=_cu(new))
    assert torch.allclose(a.float(), b.float(), atol=2.0 ** -6 if x == BF16 else 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("new", [[1, 1], [21, 20], [200, 3]])
def test_attention_exact_mode_never_reads_what_is_not_seen(new, n_q, n_kv, hd):
    """the same on an fp32 cache: what lies past the lengths and on other pages may be anything"""
    lens, prefix = [new[0] + 4, new[1] + 13], 45
    cache = Cache(lens, 16, n_kv, hd, F32, prefix=prefix, seed=5)
    seen = torch.zeros(cache.k.shape[0], 16, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for t in range(n):
            seen[cache.table[b, t // 16], t % 16] = True
    for t in range(prefix):
        seen[cache.prefix[t // 16], t % 16] = True
    q = torch.randn(sum(new), n_q, hd, device=DEV)
    want, tol = attention64(q, cache, lens, new, n_q, hd ** -0.5, False)
    hidden = (~seen)[:, None, :, None].expand_as(cache.k)
    for junk in (math.nan, math.inf, -math.inf, 3e38):
        cache.k[hidden], cache.v[hidden] = junk, junk
        check(paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=prefix, cu_rows=_cu(new)), want, tol, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n_kv,hd", [(2, 64), (1, 128)])
def test_attention_exact_mode_nonsense_row_offsets_end_in_bounds(n_kv, hd):
    cache = Cache([40, 40, 40, 40], 16, n_kv, hd, F32, prefix=20)
    q = torch.randn(90, 4, hd, device=DEV)
    for cu in ([0, 9, -4, 2 ** 31 - 1, 40], [50, 60, 70, 80, 90], [4, 3, 2, 1, 0], [0, 90, 90, 90, 90]):
        paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=20, cu_rows=torch.tensor(cu, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
    cache.lens.fill_(2 ** 31 - 1)
    paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=20, cu_rows=_cu([60, 10, 10, 10]))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_attention_nonsense_row_offsets_end_in_bounds():
    cache = Cache([40, 40, 40, 40], 16, 2, 64, BF16, prefix=20)
    q = torch.randn(40, 4, 64, device=DEV).bfloat16()
    for cu in ([0, 9, -4, 2 ** 31 - 1, 40], [50, 60, 70, 80, 90], [4, 3, 2, 1, 0], [-2 ** 31, 2 ** 31 - 1, 0, 0, 2], [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]):
        paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=20, cu_rows=torch.tensor(cu, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
    cache.lens.fill_(2 ** 31 - 1)
    paged_prefix_attention(q[:4], *cache.args(), prefix_table=cache.prefix, prefix_len=20)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_attention_visible_nan_and_infinity_stay_in_their_rows():
    """a NaN key, or a NaN / infinite value, that one sequence sees reaches that sequence's rows and no other"""
    cache = Cache([30, 30, 30], 16, 2, 64, BF16, prefix=10)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    run = lambda: paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=10)  # noqa: E731
    clean = run()
    cache.v[cache.table[1, 0].long(), :, 3] = math.nan
    got = run()
    assert bool(got[1].isnan().all()) and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    cache.v[cache.table[1, 0].long(), :, 3] = 1.0
    cache.k[cache.table[1, 0].long(), :, 3] = math.nan
    got = run()
    assert bool(got[1].isnan().all()) and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.gpu
def test_attention_and_append_past_32_bit_offsets():
    """a cache whose last page starts more than 2^32 elements in"""
    n_pages, page = 2 ** 32 // (128 * 2 * 64) + 2, 128
    k = torch.zeros(n_pages, 2, page, 64, dtype=BF16, device=DEV)
    v = torch.zeros_like(k)
    small = Cache([100], page, 2, 64, BF16, spare=0)
    k[-1], v[-1] = small.k[0], small.v[0]
    table = torch.tensor([[n_pages - 1]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, 64, device=DEV).bfloat16()
    # (against the 64-bit result: how the work is cut, and with it the order of sums, goes by the table's width)
    want, tol = attention64(q, small, [100], [1], 4, 0.125, True)
    check(paged_prefix_attention(q, k, v, table, small.lens), want, tol, 0.0)
    small.prefix, small.prefix_len = small.table[0, :1], 70
    want, tol = attention64(q, small, [100], [1], 4, 0.125, True)
    check(paged_prefix_attention(q, k, v, table, small.lens, prefix_table=table[0], prefix_len=70), want, tol, 0.0)
    qkv, tab = torch.randn(1, 8 * 64, device=DEV).bfloat16(), torch.rand(128, 32, device=DEV)
    paged_rope_append(qkv, tab, tab, k, v, table, small.lens)
    paged_rope_append(qkv, tab, tab, *small.args())
    assert torch.equal(k[-1], small.k[0]) and torch.equal(v[-1], small.v[0]) and not bool(k[:1].any()) and not bool(v[n_pages // 2].any())


@pytest.mark.gpu
@pytest.mark.parametrize("x", [BF16, F32])
@pytest.mark.parametrize("prefix", [0, 40, 3000])
def test_attention_mixed_sequences(x, prefix):
    """one long text among many single tokens: every way of cutting the work meets every kind of sequence in one launch"""
    new = [1] * 20 + [45] + [1, 0, 2] + [1] * 7
    lens = [1 + (i * 53) % 190 for i in range(20)] + [60] + [700, 5, 2] + [-1, 3, 3, 900, 17, 0, 64]
    _attn_case(lens, new, 4, 2, 64, x, BF16, prefix=prefix, seed=prefix)
    _attn_case(lens, new, 2, 1, 128, x, BF16, prefix=prefix, seed=prefix + 1)
    if x == F32:
        _attn_case(lens, new, 4, 2, 64, x, F32, prefix=prefix, seed=prefix + 2)


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 2, 64), (2, 1, 128), (3, 1, 64)])
def test_attention_short_axes(x, c, n_q, n_kv, hd):
    """axes that one workgroup walks alone: a text among single tokens, more sequences behind a longer axis, one key, padding"""
    _attn_case([5, 46, 1, 30, -1, 17, 2, 44] + [3] * 20, [1, 45, 1, 1, 1, 0, 2, 1] + [1] * 20, n_q, n_kv, hd, x, c, prefix=30, seed=1)
    _attn_case([1 + (i * 37) % 190 for i in range(180)], [1] * 180, n_q, n_kv, hd, x, c, prefix=100, seed=2)
    _attn_case([1], [1], n_q, n_kv, hd, x, c, prefix=1, seed=3)
    _attn_case([0, -1, 1], [1, 1, 1], n_q, n_kv, hd, x, c, prefix=33, seed=4, cu=None)


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("lens,new,prefix", [([30, 9], [1, 1], 20), ([30, 9], [1, 1], 3000), ([200, 60], [150, 60], 100), ([2000], [1], 0)])
def test_attention_in_place_and_strided(x, c, lens, new, prefix):
    """out = q, q as the q part of wider rows, out as a slice of wider rows"""
    cache = Cache(lens, 16, 2, 64, c, prefix=prefix)
    n = sum(new)
    wide = torch.randn(n, 10, 64, device=DEV).to(x)
    q = wide[:, 1:5]
    kw = dict(prefix_table=cache.prefix, prefix_len=prefix, cu_rows=_cu(new))
    want, tol = attention64(q, cache, lens, new, 4, 0.125, x == BF16)
    into = torch.zeros(n, 7, 64, device=DEV).to(x)
    paged_prefix_attention(q, *cache.args(), out=into[:, 2:6], **kw)
    check(into[:, 2:6], want, tol, 0.0)
    assert bool((into[:, :2] == 0).all()) and bool((into[:, 6:] == 0).all())
    beside = wide[:, 5:].clone()
    paged_prefix_attention(q, *cache.args(), out=q, **kw)
    check(q, want, tol, 0.0)
    assert torch.equal(wide[:, 5:], beside)


@pytest.mark.gpu
def test_attention_same_bits_every_time():
    cache, q, out = _attn_case([700, 90, 1300], [1, 1, 1], 8, 2, 64, BF16, BF16, prefix=900, cu=None)
    for _ in range(5):
        assert torch.equal(out, paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=900))


# ---- sampling ------------------------------------------------------------------------------------------------------------
def _sample_case(x, u, **kw):
    got = sample_filtered(x.to(DEV), u.to(DEV), **{k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()})
    assert got.shape == (*x.shape[:-1], 1) and got.dtype == torch.int32
    pick = lambda k, d, i: (kw[k][i].item() if torch.is_tensor(kw.get(k)) else kw.get(k, d))  # noqa: E731
    want = [sample64(x[i], u[i].item(), pick("temperature", 1.0, i), pick("topk", 0, i), pick("top_p", 1.0, i), pick("min_p", 0.0, i)) for i in range(x.shape[0])]
    assert got[:, 0].tolist() == want


def f32(v):
    """a setting as the kernel sees it: a Python float rounded to fp32"""
    return torch.tensor(v, dtype=F32).item()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 3, 51, 63, 64, 65, 255, 257, 1000, 2051, 5000, 16385, 40001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_settings(V, dtype):
    g = torch.Generator().manual_seed(V)
    n = 12 if V < 4000 else 4
    x = (torch.randn(n, V, generator=g) * 3).to(dtype)
    u = torch.rand(n, generator=g)
    for kw in (dict(), dict(topk=min(50, V)), dict(top_p=f32(0.9)), dict(min_p=f32(0.05)), dict(temperature=f32(0.7), topk=min(20, V), top_p=f32(0.8), min_p=f32(0.02)),
               dict(temperature=0.0), dict(topk=1), dict(topk=V), dict(top_p=f32(1e-6)), dict(min_p=1.0), dict(temperature=f32(0.01)), dict(temperature=f32(50.0), top_p=f32(0.5))):
        _sample_case(x, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_settings_per_row(dtype):
    g = torch.Generator().manual_seed(9)
    n, V = 64, 777
    x, u = (torch.randn(n, V, generator=g) * 2).to(dtype), torch.rand(n, generator=g)
    T = torch.rand(n, generator=g) * 1.5
    T[::7] = 0
    _sample_case(x, u, temperature=T, topk=torch.randint(-2, 1000, (n,), generator=g, dtype=torch.int32).clamp(max=V), top_p=torch.rand(n, generator=g), min_p=torch.rand(n, generator=g) * 0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [97, 2051, 20000])
def test_sample_ties(V):
    """few distinct values: the cuts fall inside groups of equals, which stay in index order"""
    g = torch.Generator().manual_seed(V)
    n = 16 if V < 4000 else 4
    x = torch.randint(0, 4, (n, V), generator=g).float()
    x[1], x[2] = 0.0, -0.0
    x[2, ::2] = 0.0
    u = torch.rand(n, generator=g)
    for kw in (dict(topk=7), dict(topk=min(V, 300)), dict(top_p=f32(0.37)), dict(topk=min(V, 333), top_p=f32(0.61)), dict(top_p=f32(0.999)), dict(min_p=f32(0.2)), dict(topk=1), dict(temperature=0.0)):
        _sample_case(x, u, **kw)
        _sample_case(x.to(BF16), u, **kw)


@pytest.mark.gpu
def test_sample_odd_rows():
    """masked ids, NaN, infinities, denormals, the lowest finite value, huge ranges, one lone entry, nothing at all"""
    V, inf = 300, math.inf
    g = torch.Generator().manual_seed(0)
    x = torch.randn(14, V, generator=g)
    x[0, 5:] = -inf
    x[1] = -inf
    x[2] = -inf
    x[2, 123] = -3.0
    x[3, ::3] = math.nan
    x[4] = math.nan
    x[5, 10], x[5, 200] = inf, inf
    x[6] = torch.finfo(F32).min
    x[7] = torch.finfo(F32).min
    x[7, 40] = torch.finfo(F32).max
    x[8] *= 1e-44
    x[9] = -inf
    x[9, 7], x[9, 9] = inf, 0.0
    x[10] *= 1e30
    x[11] = torch.finfo(F32).min
    x[11, ::2] = -inf
    x[12, 100:] = torch.finfo(F32).min
    for kw in (dict(), dict(topk=5), dict(top_p=f32(0.5)), dict(min_p=f32(0.5)), dict(topk=200, top_p=f32(0.95), min_p=f32(0.01), temperature=f32(1.3)), dict(temperature=0.0)):
        for u in (0.0, 0.25, 0.6180339, 1 - 2.0 ** -24):
            _sample_case(x, torch.full((14,), u), **kw)


@pytest.mark.gpu
def test_sample_uniform_sweep_and_clamps():
    x = torch.tensor([[0.0, 1.0, -math.inf, 2.0, 0.5]]).repeat(1000, 1)
    u = torch.linspace(0, 1, 1001)[:1000]
    _sample_case(x, u)
    _sample_case(x, u, top_p=f32(0.6))
    got = sample_filtered(x[:4].to(DEV), torch.tensor([-1.0, 1.0, math.nan, 7.0], device=DEV))
    assert got[:, 0].tolist() == [0, 4, 0, 4]
    odd = lambda *v: torch.tensor(v, device=DEV)  # noqa: E731
    a = sample_filtered(x[:4].to(DEV), odd(0.1, 0.1, 0.99, 0.99), temperature=odd(-1.0, math.nan, math.inf, 1.0), topk=torch.tensor([0, 0, 99, 1], dtype=torch.int32, device=DEV),
                        top_p=odd(-1.0, math.nan, 2.0, 1.0), min_p=odd(2.0, math.nan, -1.0, 0.0))
    assert a[:, 0].tolist() == [3, 3, 4, 3]


@pytest.mark.gpu
def test_sample_shapes_and_strides():
    g = torch.Generator().manual_seed(1)
    big = torch.randn(6, 1001, generator=g)
    u = torch.rand(6, generator=g)
    for dtype in (F32, BF16):
        b = big.to(dtype).to(DEV)
        for view in (b[:, 1:], b[:, 3:998], b[::2, 5:], b.t().contiguous().t()[:, :77]):
            n = view.shape[0]
            assert torch.equal(sample_filtered(view, u[:n].to(DEV), top_p=0.8, topk=50), sample_filtered(view.contiguous(), u[:n].to(DEV), top_p=0.8, topk=50))
    x3 = big[:, :500].reshape(2, 3, 500).to(DEV)
    got = sample_filtered(x3, u.view(2, 3).to(DEV), min_p=0.1)
    assert got.shape == (2, 3, 1) and torch.equal(got.view(-1), sample_filtered(x3.view(6, 500), u.to(DEV), min_p=0.1).view(-1))
    one = sample_filtered(x3[0, 0], u[:1].to(DEV).view(()), temperature=0.0)
    assert one.shape == (1,) and int(one) == int(x3[0, 0].argmax())
    assert sample_filtered(x3[:0, 0], u[:0].to(DEV)).shape == (0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_large_vocabulary(dtype):
    g = torch.Generator().manual_seed(4)
    x, u = (torch.randn(3, 128256, generator=g) * 2.5).to(dtype), torch.rand(3, generator=g)
    for kw in (dict(), dict(top_p=f32(0.9)), dict(topk=50, top_p=f32(0.9)), dict(min_p=f32(0.01)), dict(topk=100000, top_p=f32(0.99))):
        _sample_case(x, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_crowded_rows(dtype):
    """what the histogram, the list and its chunks cannot hold: one outlier far from a crowd, thousands of near-equal winners side by side, few distinct
    values, a flat row, nearly everything masked"""
    g = torch.Generator().manual_seed(2)
    for V in (3000, 9000, 40000, 70001):
        x = torch.randn(6, V, generator=g)
        x[0] = x[0] * 1e-3
        x[0, 17] = 1e4
        x[1, V // 3:V // 3 + min(5000, V // 3)] += 8.0
        x[2] = torch.randint(0, 3, (V,), generator=g).float()
        x[3] = x[3] * 1e-6
        x[4, :V - 30] = -math.inf
        x[5] = -1e4
        x[5, 5:80] = torch.linspace(0, 1e-3, 75)
        x, u = x.to(dtype), torch.rand(6, generator=g)
        for kw in (dict(top_p=f32(0.9)), dict(topk=min(V, 4000), top_p=f32(0.95)), dict(topk=64), dict(topk=65, min_p=f32(0.3)), dict(min_p=f32(0.7)), dict()):
            _sample_case(x, u, **kw)


@pytest.mark.gpu
def test_sample_captured():
    """short and long rows in one graph, replayed with new inputs"""
    g = torch.Generator().manual_seed(6)
    xs = [torch.randn(3, V, generator=g).to(DEV) for V in (2051, 5000, 20011)]
    u = torch.rand(3, generator=g).to(DEV)
    run = lambda: [sample_filtered(x, u, topk=50, top_p=0.9) for x in xs] + [sample_filtered(x, u, top_p=0.7) for x in xs]  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(4):
        g.manual_seed(seed)
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=g))
        u.copy_(torch.rand(3, generator=g))
        graph.replay()
        torch.randn(1000, device=DEV).sum().item()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))


@pytest.mark.gpu
def test_python_refusals():
    c = Cache([5, 5], 16, 2, 64, BF16, prefix=16)
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    ok = lambda **k: paged_prefix_attention(k.pop("q", q), k.pop("k", c.k), k.pop("v", c.v), k.pop("table", c.table), k.pop("lens", c.lens), **k)  # noqa: E731
    ok()
    for bad in (dict(q=q.float()[:, :3]), dict(q=q[:1]), dict(q=q.half()), dict(q=q[..., :32]), dict(k=c.k.float()), dict(v=c.v[:1]), dict(table=c.table.long()), dict(lens=c.lens[:1]),
                dict(lens=c.lens.long()), dict(out=q.float()), dict(out=q[:1]), dict(cu_rows=c.lens), dict(prefix_len=5), dict(prefix_len=17, prefix_table=c.prefix),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(k=c.k.transpose(2, 3).contiguous().transpose(2, 3)), dict(scale=math.nan), dict(lens=c.lens.cpu()),
                dict(q=q.float().requires_grad_()), dict(prefix_table=c.prefix.long(), prefix_len=3)):
        with pytest.raises((ValueError, RuntimeError)):
            ok(**bad)
    with torch.no_grad():
        ok(q=q.clone().requires_grad_())
    x, u = torch.randn(2, 9, device=DEV), torch.rand(2, device=DEV)
    for bad in (dict(topk=10), dict(topk=-1), dict(top_p=0.0), dict(min_p=1.5), dict(temperature=-1.0), dict(temperature=torch.ones(3, device=DEV)), dict(topk=torch.ones(2, device=DEV)),
                dict(top_p=torch.ones(2))):
        with pytest.raises((ValueError, RuntimeError)):
            sample_filtered(x, u, **bad)
    with pytest.raises(ValueError):
        sample_filtered(x, u.double())
    with pytest.raises(ValueError):
        sample_filtered(x.half(), u)
    tab = torch.zeros(8, 32, device=DEV)
    for qkv in (torch.zeros(2, 7 * 64 + 1, device=DEV), torch.zeros(2, 4 * 64, device=DEV), torch.zeros(3, 8 * 64, device=DEV), torch.zeros(2, 8 * 64, device=DEV, dtype=torch.half)):
        with pytest.raises((ValueError, RuntimeError)):
            paged_rope_append(qkv, tab, tab, *c.args())
    with pytest.raises(ValueError):
        paged_rope_append(torch.zeros(2, 8 * 64, device=DEV), tab, tab[:, :16], *c.args())


@pytest.mark.gpu
def test_numbers_and_lonely_strides():
    """settings are whole numbers where they count something; the stride of a dimension of size one is never looked at"""
    x, u = torch.randn(2, 9, device=DEV), torch.rand(2, device=DEV)
    for bad, kind in ((dict(topk=2.0), TypeError), (dict(topk=1 << 70), ValueError), (dict(topk=1 << 31), ValueError), (dict(top_p="1"), TypeError), (dict(min_p=None), TypeError)):
        with pytest.raises(kind):
            sample_filtered(x, u, **bad)
    c = Cache([5], 16, 1, 64, F32)
    q = torch.randn(1, 4, 64, device=DEV)
    odd = lambda t, *d: t.as_strided(t.shape, [7 if i in d else n for i, n in enumerate(t.stride())])  # noqa: E731
    want = paged_prefix_attention(q, c.k, c.v, c.table, c.lens)
    assert torch.equal(paged_prefix_attention(odd(q, 0), odd(c.k, 1), odd(c.v, 1), odd(c.table, 0), c.lens), want)
    assert torch.equal(sample_filtered(odd(x[:1], 0), u[:1]), sample_filtered(x[:1], u[:1]))
    qkv, tab = torch.randn(1, 6 * 64, device=DEV), torch.rand(8, 32, device=DEV)
    assert torch.equal(paged_rope_append(odd(qkv, 0), tab, tab, odd(c.k, 1), c.v, c.table, c.lens), paged_rope_append(qkv, tab, tab, c.k, c.v, c.table, c.lens))


# ---- the three as one serving step -----------------------------------------------------------------------------------------
class Step:
    """One decode step of a small model head: packed projection rows -> append -> attention -> logits -> sampled token."""

    def __init__(self, x=BF16, c=BF16, seed=0, b=5, off=40, room=32):
        self.n_q, self.n_kv, self.hd, self.V, self.off, self.b = 8, 2, 64, 301, off, b
        self.cache = Cache([room] * b, 16, 2, 64, c, prefix=off, seed=seed)
        self.start = torch.tensor([3, 17, 1, 9, -1][:b], dtype=torch.int32, device=DEV)
        self.cache.lens.copy_(self.start)
        g = torch.Generator().manual_seed(seed + 5)
        self.emb = torch.randn(self.V, 12 * 64, generator=g).to(x).to(DEV)
        self.head = (torch.randn(8 * 64, self.V, generator=g) * 0.3).to(x).to(DEV)
        ang = torch.arange(off + room, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64))
        self.cos, self.sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
        self.tok = torch.zeros(b, 1, dtype=torch.int32, device=DEV)
        self.u = torch.zeros(b, device=DEV)
        self.out = torch.zeros(b, 8, 64, dtype=x, device=DEV)
        self.set = dict(temperature=0.8, topk=40, top_p=0.9, min_p=0.01)

    def run(self):
        qkv = self.emb[self.tok[:, 0].long()]
        self.cache.lens.copy_(torch.where(self.cache.lens < 0, self.cache.lens, self.cache.lens + 1))
        self.q = paged_rope_append(qkv, self.cos, self.sin, *self.cache.args(), pos_offset=self.off)
        paged_prefix_attention(self.q, *self.cache.args(), prefix_table=self.cache.prefix, prefix_len=self.off, out=self.out)
        self.logits = self.out.flatten(1).float() @ self.head.float()
        self.tok.copy_(sample_filtered(self.logits, self.u, **self.set))
        return self.tok


def _plain_step(s, kv64, tok, u, lens):
    """the same step in 64 bits on its own cache; returns (attention, logits) of the live rows"""
    x = s.emb[tok.long()].double().view(s.b, 12, 64)
    want = torch.zeros(s.b, 8, 64, dtype=torch.float64, device=DEV)
    for b in range(s.b):
        if lens[b] < 0:
            continue
        slot = lens[b] - 1
        cs, sn = s.cos[s.off + slot].double(), s.sin[s.off + slot].double()
        lo, hi = x[b, :10, :32], x[b, :10, 32:]
        y = torch.cat((lo * cs - hi * sn, hi * cs + lo * sn), 1)
        kv64[b][0].append(y[8:].clone())
        kv64[b][1].append(x[b, 10:].clone())
        k, v = (torch.cat((p, torch.stack(o, 1)), 1) for p, o in zip(kv64["prefix"], kv64[b]))
        p = torch.softmax(y[:8].view(2, 4, 64) @ k.transpose(1, 2) / 8.0, -1)
        want[b] = (p @ v).reshape(8, 64)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(F32, F32), (BF16, BF16)])
def test_serving_steps_match_the_plain_step(x, c):
    s = Step(x, c)
    flat = lambda z: z.double().transpose(0, 1).reshape(2, -1, 64)  # noqa: E731
    kv = {"prefix": [flat(z[s.cache.prefix.long()])[:, :s.off] for z in (s.cache.k, s.cache.v)]}
    for b in range(s.b):
        n = max(0, int(s.start[b]))
        kv[b] = [[r for r in flat(z[s.cache.table[b, :2].long()])[:, :n].unbind(1)] for z in (s.cache.k, s.cache.v)]
    g = torch.Generator().manual_seed(3)
    # fp32: a handful of roundings of values near 1; bf16: q, k and the result each rounded once (2^-8), a score of magnitude up to about 30 moves by 30 * 2 * 2^-8
    tol = 2e-4 if x == F32 else 0.25
    for step in range(6):
        tok, lens = s.tok[:, 0].clone(), (s.cache.lens + (s.cache.lens >= 0)).tolist()
        s.u.copy_(torch.rand(s.b, generator=g))
        s.run()
        want = _plain_step(s, kv, tok, s.u, lens)
        assert float((s.out.double() - want).abs().max()) < tol
        for b in range(s.b):        # the token is the exact draw from the step's own logits
            assert int(s.tok[b]) == sample64(s.logits[b].cpu(), s.u[b].item(), f32(0.8), 40, f32(0.9), f32(0.01))


@pytest.mark.gpu
def test_serving_step_captured_and_replayed():
    """two graphs of the same step on states of their own, replayed in turn with eager work between, against eager runs"""
    def steps(states, runs, n):
        out = []
        g = torch.Generator().manual_seed(8)
        for _ in range(n):
            for s, r in zip(states, runs):
                s.u.copy_(torch.rand(s.b, generator=g))
                r()
                torch.randn(1000, device=DEV).sum().item()
                out.append((s.tok.clone(), s.out.clone(), s.cache.k.clone()))
        return out
    eager = [Step(seed=1), Step(seed=2, off=300)]
    want = steps(eager, [s.run for s in eager], 5)
    states, graphs = [Step(seed=1), Step(seed=2, off=300)], []
    for s in states:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run()
        fresh = Step(seed=1 if not graphs else 2, off=s.off)
        s.cache.lens.copy_(fresh.cache.lens)
        s.cache.k.copy_(fresh.cache.k)
        s.cache.v.copy_(fresh.cache.v)
        s.tok.zero_()
        s.out.zero_()
        graphs.append(graph)
    got = steps(states, [g.replay for g in graphs], 5)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_operators_run_on_the_current_stream():
    """work queued on a side stream behind a slow kernel: the operators see its results, i.e. they run on that stream"""
    s, ref = Step(seed=4), Step(seed=4)
    ref.run()
    emb = s.emb.clone()
    s.emb.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slow = torch.randn(4096, 4096, device=DEV)
        for _ in range(20):
            slow = slow @ slow * 1e-3
        s.emb.copy_(emb)
        s.run()
    side.synchronize()
    assert torch.equal(s.tok, ref.tok) and torch.equal(s.out, ref.out) and torch.equal(s.cache.k, ref.cache.k)
