"""The stand-alone operators of include/csm_ops.h where they are used otherwise than in test_paged_ops.py: roundings of single steps, settings and
sizes at the end of their ranges, calls that have to be refused.  Tolerances count roundings (half a step: fp32 2^-24, bf16 2^-8)."""
import ctypes as C
import math

import pytest
import torch

from csm_hf_amd import ops, paged_prefix_attention, paged_rope_append, sample_filtered
from test_paged_ops import BF16, Cache, DEV, F32, HALF, _cu, _paged_args, _sample_case, attention64, check, f32


# ---- attention -----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("b,n_q,n_kv,hd,prefix,longest", [(40, 8, 2, 64, 900, 200), (130, 4, 1, 64, 300, 40), (40, 4, 2, 128, 900, 100), (9, 8, 2, 64, 700, 300)])
def test_attention_weights_of_decode_batches_are_not_rounded_to_bf16(b, n_q, n_kv, hd, prefix, longest):
    """One new token per sequence behind a shared prefix: beside the one rounding of the result, a weight is off by 2^-15 at most (a truncated bf16
    piece leaves less than 2^-7 of it, and of that the second piece is off by half a step)."""
    lens = [max(1, longest - (i * 37) % longest) for i in range(b)]
    cache = Cache(lens, 16, n_kv, hd, BF16, prefix=prefix, seed=b)
    q = torch.randn(b, n_q, hd, generator=torch.Generator().manual_seed(b)).to(BF16).to(DEV)
    got = paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=prefix)
    want, tol = attention64(q, cache, lens, [1] * b, n_q, hd ** -0.5, False)
    mag, _ = attention64(q, _abs_v(cache), lens, [1] * b, n_q, hd ** -0.5, False)
    check(got, want, tol + mag * 2.0 ** -15 + want.abs() * HALF[BF16], 0.0)


def _abs_v(cache):
    other = object.__new__(Cache)
    other.__dict__.update(cache.__dict__, v=cache.v.abs())
    return other


@pytest.mark.gpu
@pytest.mark.parametrize("x,c", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("new", [[1, 1], [1, 40]])
@pytest.mark.parametrize("scale", [0.0, 5e-38, -5e-38, 1e-44])
def test_attention_smallest_scales(scale, new, x, c):
    """scores near 1e37 under scales below 1e-37: a plain mean for a scale of 0, the softmax of the scaled scores for the others"""
    lens, prefix = [90, 300], 70
    cache = Cache(lens, 16, 2, 64, c, prefix=prefix, seed=3)
    cache.k *= 1e18
    q = (torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(3)) * 1e18).to(x).to(DEV)
    got = paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=prefix, cu_rows=_cu(new), scale=scale)
    s = float(torch.tensor(scale, dtype=F32))
    want, tol = attention64(q, cache, lens, new, 4, s, x == BF16)
    # scale * log2(e) is a denormal number of steps of 2^-149, off by one of them: 2^-149 times scores of at most 64 * 5e18 * 5e18 is 2^-18
    check(got, want, tol + 2 * 2.0 ** -18, 0.0)


def test_scales_that_are_not_finite_in_powers_of_two_are_refused():
    lib = ops.load_ops_library()
    a = ops.AttentionArgs(q=1 << 24, out=1 << 25, q_stride=256, out_stride=256, x_dtype=1, n_q=4, scale=3e38, workspace=1 << 28, workspace_bytes=1 << 27)
    _paged_args(a.c)
    assert lib.csm_ops_paged_prefix_attention(bytes(a), None) == -1


# ---- sampling ------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,low,first,u,how", [
    (*row, how) for row in ((2 ** 21, -29.75, True, 1 - 2.0 ** -24), (2 ** 21, -31.0, False, 2.0 ** -27), (2 ** 18 + 1, -30.0, False, 2.0 ** -27), (2 ** 17, -30.0, False, 2.0 ** -28))
    for how in ("all", "top_p", "topk", "min_p") if how != "top_p" or row[0] == 2 ** 21])     # (shorter tails are less than the largest top_p below 1 leaves out)
def test_sample_flat_tail_of_the_longest_rows(V, low, first, u, how, dtype):
    """One dominant value and a flat tail of V - 1 others that holds 2^-27 to 2^-22 of the mass, with a target inside it.  A weight is off by 2^-52 of the
    largest at most (2^-49 where the row's chunks are drawn from): with x = (u (1 + n w) - 1) / w, or u (1 + n w) / w, and the tail's mass above 1 - u (or u),
    V of these roundings move x by at most V 2^-52 / w places, a nucleus that cuts the tail by as much again."""
    x = torch.full((1, V), low)
    x[0, 0 if first else V - 1] = 0.0
    w, n = math.exp(low), V - 1
    kw = {"all": dict(), "top_p": dict(top_p=1 - 2.0 ** -24), "topk": dict(topk=V - V // 8), "min_p": dict(min_p=w / 2)}[how]
    if how == "topk":
        n = kw["topk"] - 1
    if how == "top_p":
        n = min(n, max(0, math.ceil((kw["top_p"] * (1 + n * w) - 1) / w)))
    want = u * (1 + n * w)
    place = (want - 1) / w + 1 if first else want / w        # tail entries in front of the token
    got = int(sample_filtered(x.to(dtype).to(DEV), torch.tensor([u], device=DEV), **kw))
    assert 0 < place < n
    assert abs(got - place) <= 2 * (V * 2.0 ** -52 + (8192 * 2.0 ** -49 if how == "all" else 0)) / w + 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,skew", [(16385, 0), (20000, 0), (32000, 0), (50257, 0), (65000, 0), (128256, 2.0), (128256, 8.0)])
def test_sample_long_rows_of_every_length(V, skew, dtype):
    """lengths at which a chunk lists a large part of its entries, and rows whose large values all stand in one chunk"""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(3, V, generator=g) * 2.5
    x[:, 8192:16384] += skew
    u = torch.rand(3, generator=g)
    for kw in (dict(top_p=f32(0.9)), dict(min_p=f32(0.05)), dict(topk=4000, top_p=f32(0.95))):
        _sample_case(x.to(dtype), u, **kw)


def _us(f):
    """least time of a call among others, in microseconds"""
    f()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            f()
    a, b, best = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True), math.inf
    for _ in range(8):
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 100)
    return best


@pytest.mark.gpu
@pytest.mark.parametrize("V,skew", [(16385, 0), (20000, 0), (32000, 0), (50257, 0), (128256, 3.0)])
def test_sample_long_rows_do_not_stream(V, skew):
    """64 rows whose nucleus fits the list take about the time of 64 rows of 128 256 spread evenly (20 percent more at most; a search that streams over the
    row takes four times as much and more)"""
    g = torch.Generator().manual_seed(0)
    make = lambda n: (torch.randn(64, n, generator=g) * 2.5).to(BF16).to(DEV)  # noqa: E731
    even, x, u = make(128256), make(V), torch.rand(64, generator=g).to(DEV)
    x[:, :8192] += skew
    assert _us(lambda: sample_filtered(x, u, temperature=0.9, top_p=0.9)) < 2.5 * _us(lambda: sample_filtered(even, u, temperature=0.9, top_p=0.9))


# ---- refusals --------------------------------------------------------------------------------------------------------------
def _calls():
    """each operator as a function of one of its tensors, that tensor, and the words its name has in a refusal"""
    c = Cache([5, 5], 16, 2, 64, F32, prefix=16)
    q, qkv, tab = torch.randn(2, 4, 64, device=DEV), torch.randn(2, 8 * 64, device=DEV), torch.rand(32, 32, device=DEV)
    x, u = torch.randn(2, 99, device=DEV), torch.rand(2, device=DEV)
    return [(lambda t: paged_prefix_attention(t, *c.args()), q), (lambda t: paged_prefix_attention(q, t, c.v, c.table, c.lens), c.k),
            (lambda t: paged_rope_append(t, tab, tab, *c.args()), qkv), (lambda t: paged_rope_append(qkv, tab, t, *c.args()), tab),
            (lambda t: sample_filtered(t, u), x), (lambda t: sample_filtered(x, u, temperature=t), u)]


@pytest.mark.gpu
def test_tangents_transforms_sparse_tensors_and_negated_views_are_refused():
    import torch.autograd.forward_ad as fwd
    for f, t in _calls():
        f(t)
        with fwd.dual_level():
            dual = fwd.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="tangent"):
                f(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                f(dual)
            f(fwd.unpack_dual(dual).primal)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))
        with pytest.raises(RuntimeError, match="function transform"):
            torch.func.vmap(f)(t[None])
        with pytest.raises(ValueError, match="dense"):
            f(t.to_sparse())
        with pytest.raises(ValueError, match="negated"):
            f(torch._neg_view(t))
        f(t)


@pytest.mark.gpu
def test_writes_into_tensors_saved_for_a_backward_pass_are_noticed():
    """autograd raises instead of using a cache or an output that a call has changed since"""
    c = Cache([5, 5], 16, 2, 64, F32)
    qkv, tab = torch.randn(2, 8 * 64, device=DEV), torch.rand(32, 32, device=DEV)
    q_out, out = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, 4, 64, device=DEV)
    append = lambda: paged_rope_append(qkv, tab, tab, *c.args(), q_out=q_out)  # noqa: E731
    attend = lambda: paged_prefix_attention(q_out, *c.args(), out=out)  # noqa: E731
    for saved, call in ((c.k, append), (c.v, append), (q_out, append), (out, attend)):
        w = torch.ones_like(saved, requires_grad=True)
        y = (w * saved).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    w = torch.ones_like(q_out, requires_grad=True)
    y = (w * q_out).sum()
    attend()                                              # reads q and the cache
    y.backward()
    assert torch.equal(w.grad, q_out)
    with torch.inference_mode():
        k = c.k.clone()
    paged_rope_append(qkv, tab, tab, k, c.v, c.table, c.lens)


@pytest.mark.parametrize("refused,over", [
    (True, dict(rows=1 << 24, n_seqs=1 << 24)), (False, dict(rows=1 << 22, n_seqs=1 << 22)),
    # many short sequences of 31 query rows a kv-head: the partial results' launch is the largest
    (True, dict(rows=2200000, n_seqs=2200000, n_q=31, n_kv=1, prefix_table=1 << 26, prefix_pages=2, prefix_len=32)),
    (False, dict(rows=2100000, n_seqs=2100000, n_q=31, n_kv=1, prefix_table=1 << 26, prefix_pages=2, prefix_len=32))])
def test_attention_launches_of_2_32_threads_are_refused(refused, over):
    """before anything is launched: sizes that fit are only asked for their workspace"""
    lib, need = ops.load_ops_library(), C.c_size_t()
    a = ops.AttentionArgs(q=1 << 24, out=1 << 25, q_stride=31 * 64 + 64, out_stride=31 * 64 + 64, x_dtype=0, n_q=4, scale=0.125, workspace=1 << 28, workspace_bytes=1 << 60)
    _paged_args(a.c, **over)
    for k, v in over.items():
        if not hasattr(a.c, k):
            setattr(a, k, v)
    assert lib.csm_ops_paged_attention_workspace(bytes(a), C.byref(need)) == (-3 if refused else 0)
    if refused:
        assert lib.csm_ops_paged_prefix_attention(bytes(a), None) == -3 and b"one launch" in lib.csm_ops_last_error()


@pytest.mark.parametrize("V,rows", [(1000, 1 << 24), (4096, 1 << 24), (4097, 1 << 22), (16384, 1 << 22), (16385, 1 << 22), (131072, 1 << 20), (1 << 21, 1 << 16)])
def test_sample_launches_of_2_32_threads_are_refused(V, rows):
    lib, need = ops.load_ops_library(), C.c_size_t()
    a = ops.SampleArgs(logits=1 << 20, logits_stride=0, x_dtype=0, rows=rows, V=V, uniform=1 << 21, temperature=1.0, top_p=0.5, out=1 << 22, workspace=1 << 30, workspace_bytes=1 << 60)
    assert lib.csm_ops_sample_workspace(bytes(a), C.byref(need)) == -3
    assert lib.csm_ops_sample_filtered(bytes(a), None) == -3 and b"one launch" in lib.csm_ops_last_error()
    a.rows -= 1
    assert lib.csm_ops_sample_workspace(bytes(a), C.byref(need)) == 0


def _append_args(**over):
    a = ops.RopeAppendArgs(qkv=1 << 24, q_out=1 << 25, qkv_stride=384, q_out_stride=128, x_dtype=1, n_q=2, cos=1 << 26, sin=1 << 27, rope_positions=64)
    _paged_args(a.c, **over)
    return a


# (4 pages of 2 heads of 16 slots of 64 bf16 values)
@pytest.mark.parametrize("over", [
    dict(k_page_stride=64), dict(k_page_stride=1024), dict(v_head_stride=512), dict(v_page_stride=1984), dict(k_page_stride=1024, k_head_stride=1024), dict(k_slot_stride=128),
    dict(v=1 << 20), dict(v=(1 << 20) + 2048), dict(v=(1 << 20) + 2 * 2 * 2048, n_pages=3), dict(k=(1 << 21) + 64), dict(v=1 << 20, v_page_stride=4096)])
def test_append_refuses_caches_whose_slots_overlap(over):
    assert ops.load_ops_library().csm_ops_paged_rope_append(bytes(_append_args(**over)), None) == -1 and b"overlap" in ops.load_ops_library().csm_ops_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("make", [
    lambda n: torch.zeros(n, 2, 2, 16, 64, device=DEV).unbind(1), lambda n: torch.zeros(2, n, 2, 16, 64, device=DEV).unbind(0), lambda n: torch.zeros(n, 2, 16, 2, 64, device=DEV).unbind(3),
    lambda n: torch.zeros(n, 16, 2, 2, 64, device=DEV).permute(3, 0, 2, 1, 4).unbind(0), lambda n: torch.zeros(n, 2, 16, 128, device=DEV).split(64, 3), lambda n: torch.zeros(2 * n, 2, 16, 64, device=DEV).unflatten(0, (n, 2)).unbind(1)[::-1],
    lambda n: torch.zeros(2, n, 16, 128, device=DEV).permute(1, 0, 2, 3).split(64, 3), lambda n: (torch.zeros(n, 2, 16, 64, device=DEV), torch.zeros(n, 16, 2, 64, device=DEV).transpose(1, 2))])
def test_append_into_one_buffer_for_k_and_v(make):
    """every order of pages, heads, slots, and of K beside V, that keeps the slots apart"""
    c = Cache([9, 33, 1], 16, 2, 64, F32, seed=2)
    k, v = make(c.k.shape[0])
    qkv, tab = torch.randn(43, 8 * 64, device=DEV), torch.rand(33, 32, device=DEV)
    for t in (c.k, c.v):
        t.zero_()
    cu = _cu([9, 33, 1])
    assert torch.equal(paged_rope_append(qkv, tab, tab, k, v, c.table, c.lens, cu_rows=cu), paged_rope_append(qkv, tab, tab, *c.args(), cu_rows=cu))
    assert torch.equal(k, c.k) and torch.equal(v, c.v)


@pytest.mark.gpu
def test_append_refuses_one_tensor_for_both_caches():
    c = Cache([5], 16, 2, 64, F32)
    qkv, tab = torch.randn(1, 8 * 64, device=DEV), torch.rand(32, 32, device=DEV)
    for k, v in ((c.k, c.k), (c.k[:-1], c.k[1:]), (c.k[:1].expand(3, 2, 16, 64), c.v[:3])):
        with pytest.raises(RuntimeError, match="overlap"):
            paged_rope_append(qkv, tab, tab, k, v, c.table, c.lens)


def test_c_entries_take_structures_by_reference():
    lib, need = ops.load_ops_library(), C.c_size_t()
    s = ops.SampleArgs(logits=1 << 20, logits_stride=20000, rows=2, V=20000, uniform=1 << 21, temperature=1.0, top_p=0.5, out=1 << 22)
    assert lib.csm_ops_sample_workspace(C.byref(s), C.byref(need)) == 0 and need.value > 0
    assert lib.csm_ops_sample_filtered(C.byref(s), None) == -3                 # no workspace
    assert lib.csm_ops_paged_rope_append(C.byref(_append_args(k_slot_stride=60)), None) == -1
    a = ops.AttentionArgs(q=1 << 24, out=1 << 25, q_stride=256, out_stride=256, x_dtype=1, n_q=4, scale=0.125)
    _paged_args(a.c)
    assert lib.csm_ops_paged_attention_workspace(C.byref(a), C.byref(need)) == 0


@pytest.mark.gpu
def test_c_entry_on_a_structure():
    lib = ops.load_ops_library()
    x, u, out = torch.randn(3, 500, device=DEV), torch.rand(3, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    s = ops.SampleArgs(logits=x.data_ptr(), logits_stride=500, x_dtype=0, rows=3, V=500, uniform=u.data_ptr(), temperature=0.8, top_p=0.9, topk=50, out=out.data_ptr())
    assert lib.csm_ops_sample_filtered(C.byref(s), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, sample_filtered(x, u, temperature=0.8, top_p=0.9, topk=50)[:, 0])
