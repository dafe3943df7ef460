"""Measured cases of the paged-cache serving operators: `paged_rope_append` (rotary embedding + append into a paged KV cache),
`paged_prefix_attention` (attention over own pages and a prefix that the whole batch shares) and `sample_filtered` (temperature / top-k /
top-p / min-p sampling from given uniforms).  `run` computes them in plain torch, or calls the framework's operators where `own` is true."""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    A, T, S = "append", "attention", "sample"
    return [
        # one utterance, one new frame: a launch and nothing else (csm-1b backbone heads)
        dict(name="append_b1", op=A, b=1, t=1, own=600, off=512, nq=32, nkv=8, hd=64, x="bf16", c="bf16", page=64, idle=0),
        # a serving batch, one frame each, fp32 activations into the default bf16 cache; two idle rows of the padded batch
        dict(name="append_b96_f32", op=A, b=96, t=1, own=1999, off=512, nq=32, nkv=8, hd=64, x="f32", c="bf16", page=16, idle=2),
        # the texts of 16 joining utterances behind the shared voice, ragged
        dict(name="append_ragged", op=A, b=16, t=181, own=181, off=1024, nq=32, nkv=8, hd=64, x="bf16", c="bf16", page=32, idle=0),
        # a long context of the 128-wide decoder heads, exact mode (fp32 cache)
        dict(name="append_long_f32", op=A, b=4, t=2048, own=2048, off=0, nq=8, nkv=2, hd=128, x="f32", c="f32", page=128, idle=0),
        # one utterance: 512 frames of voice, its own frames behind it
        dict(name="attn_b1", op=T, b=1, t=1, own=131, off=512, nq=32, nkv=8, hd=64, x="bf16", c="bf16", page=64, idle=0),
        # sixteen rows in the exact mode (fp32 activations and cache)
        dict(name="attn_b16_f32", op=T, b=16, t=1, own=333, off=512, nq=32, nkv=8, hd=64, x="f32", c="f32", page=16, idle=1),
        # a serving batch of 64 rows behind one long voice prompt, 128-wide heads, fp32 activations over the default bf16 cache
        dict(name="attn_b64_hd128", op=T, b=64, t=1, own=777, off=2048, nq=8, nkv=2, hd=128, x="f32", c="bf16", page=32, idle=3),
        # the largest batch late in its generation: own caches dominate
        dict(name="attn_b128_long", op=T, b=128, t=1, own=2048, off=4096, nq=32, nkv=8, hd=64, x="bf16", c="bf16", page=64, idle=0),
        # texts of 16 joining utterances over the shared voice: many query rows per sequence
        dict(name="attn_ragged", op=T, b=16, t=181, own=181, off=2048, nq=32, nkv=8, hd=64, x="bf16", c="bf16", page=32, idle=0),
        # one codebook of one utterance: the reference's usual call plus a nucleus
        dict(name="sample_b1", op=S, rows=1, v=2051, x="f32", mode="all", masked=0),
        # the same for a large batch, every row with its own settings
        dict(name="sample_b512", op=S, rows=512, v=2051, x="f32", mode="rows", masked=1),
        # a text vocabulary, nucleus only: the mass of the whole row counts
        dict(name="sample_text", op=S, rows=64, v=128256, x="bf16", mode="top_p", masked=0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "sample"))
    if op == "sample":
        v = rng.choice((51, 2051, 2051, 128256, _log(rng, 40, 60000)))
        rows = _log(rng, 1, max(1, min(2048, 64 * 128256 // v)))
        return dict(op=op, rows=rows, v=v, x=rng.choice(("f32", "bf16")), mode=rng.choice(("all", "rows", "top_p", "min_p", "topk", "none")), masked=rng.randrange(2))
    nq, nkv, hd = rng.choice(((32, 8, 64), (8, 2, 128), (4, 1, 64), (2, 1, 128), (12, 4, 64), (6, 6, 128)))
    x, c = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")))
    page = rng.choice((8, 16, 32, 64, 128))
    off = rng.choice((0, _log(rng, 1, 4096)))
    if rng.random() < 0.6:      # one new frame per row
        b, t, longest = _log(rng, 1, 128), 1, _log(rng, 1, 2048)
        longest = max(1, min(longest, 128 * 2048 * 512 * 2 // (b * nkv * hd * (4 if c == "f32" else 2))))      # bytes of the largest listed caches
    else:                       # joining texts / contexts
        b = _log(rng, 1, 16)
        t = _log(rng, 2, 181 if op == "attention" else 512)
        longest = t + rng.choice((0, _log(rng, 1, 300)))
        off = min(off, 2048)
    return dict(op=op, b=b, t=t, own=longest, off=off, nq=nq, nkv=nkv, hd=hd, x=x, c=c, page=page, idle=rng.choice((0, 0, min(b - 1, 2))))


def _shape(case):
    """New rows and own length (new rows included) of every sequence: lists of b numbers.  The last `idle` sequences are padding (length -1)."""
    b, t, n = case["b"], case["t"], case["own"]
    new = [t if t == 1 else max(1, t - (i * 41) % (t // 2 + 1)) for i in range(b)]
    lens = [max(new[i], n - (i * 67) % (n // 2 + 1)) for i in range(b)]
    lens = [-1 if i >= b - case["idle"] else lens[i] for i in range(b)]
    return new, lens


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 11)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if case["op"] == "sample":
        rows, v = case["rows"], case["v"]
        x = rand(rows, v) * 2.5
        if case["masked"]:      # ids that a grammar or the codec forbids
            x[:, 3::7] = -math.inf
        s = dict(case=case, logits=x.to(DT[case["x"]]), u=torch.rand(rows, generator=g, device=dev))
        r = lambda lo, hi: torch.rand(rows, generator=g, device=dev) * (hi - lo) + lo  # noqa: E731
        mode = case["mode"]
        s["set"] = dict(temperature=0.9, topk=0, top_p=1.0, min_p=0.0)
        if mode in ("all", "topk"):
            s["set"]["topk"] = min(50, v)
        if mode in ("all", "top_p"):
            s["set"]["top_p"] = 0.9
        if mode in ("all", "min_p"):
            s["set"]["min_p"] = 0.05
        if mode == "rows":
            k = (torch.rand(rows, generator=g, device=dev) * min(200, v)).to(torch.int32)
            s["set"] = dict(temperature=r(0.5, 1.5), topk=k, top_p=r(0.3, 1.0), min_p=r(0.0, 0.2))
            s["set"]["temperature"][::9] = 0.0
        return s
    new, lens = _shape(case)
    b, page, nq, nkv, hd = case["b"], case["page"], case["nq"], case["nkv"], case["hd"]
    per = [max(1, -(-max(n, 0) // page)) for n in lens]
    width = max(per) + 1
    n_prefix = -(-case["off"] // page) if case["op"] == "attention" else 0
    n_pages = sum(per) + n_prefix + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.full((b, width), -1, dtype=torch.int32)
    at = n_prefix
    for i in range(b):
        table[i, :per[i]] = order[at:at + per[i]]
        at += per[i]
    cu = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32)
    rows = int(cu[-1])
    s = dict(case=case, table=table.to(dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev), prefix=order[:n_prefix].to(dev),
             cu=None if case["t"] == 1 else cu.to(dev), rows=rows, width=width)
    s["k"], s["v"] = (rand(n_pages, nkv, page, hd).to(DT[case["c"]]) for _ in range(2))
    if case["op"] == "append":
        s["qkv"] = rand(rows, (nq + 2 * nkv) * hd).to(DT[case["x"]])
        inv = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
        ang = torch.arange(case["off"] + case["own"], dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float().to(dev), ang.sin().float().to(dev)
        s["out"] = torch.zeros(rows, nq, hd, dtype=DT[case["x"]], device=dev)
    else:
        s["q"] = (rand(rows, nq, hd) * 1.5).to(DT[case["x"]])
        s["out"] = torch.zeros_like(s["q"])
    return s


def _rows(s):
    """Sequence, place among its new rows and cache slot of every row; slot -1 for the rows of padding."""
    r = torch.arange(s["rows"], device=s["lens"].device)
    if s["cu"] is None:
        seq, t, new = r, torch.zeros_like(r), torch.ones_like(r)
    else:
        cu = s["cu"].long()
        seq = torch.searchsorted(cu, r, right=True) - 1
        t, new = r - cu[seq], cu[seq + 1] - cu[seq]
    n = s["lens"].long()[seq]
    return seq, t, torch.where(n < 0, -1, n - new + t)


def _append_plain(s):
    c = s["case"]
    nq, nkv, hd, page = c["nq"], c["nkv"], c["hd"], c["page"]
    seq, _, slot = _rows(s)
    live = slot >= 0
    pos = (slot + c["off"]).clamp(min=0)
    x = s["qkv"].float().view(s["rows"], nq + 2 * nkv, hd)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    lo, hi = x[:, :nq + nkv, :hd // 2], x[:, :nq + nkv, hd // 2:]
    rot = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)
    s["out"].copy_(torch.where(live[:, None, None], rot[:, :nq].to(s["out"].dtype), s["out"]))
    at = slot.clamp(min=0)
    pages = torch.where(live, s["table"].long()[seq, at // page], s["k"].shape[0])
    grow = lambda z: torch.cat((z, z[:1]))  # noqa: E731  one more page takes what the padding would write
    for_k, for_v = grow(s["k"]), grow(s["v"])
    for_k[pages, :, at % page] = rot[:, nq:].to(for_k.dtype)
    for_v[pages, :, at % page] = x[:, nq + nkv:].to(for_v.dtype)
    s["k"].copy_(for_k[:-1])
    s["v"].copy_(for_v[:-1])
    return s["out"], s["k"], s["v"]


def _attention_plain(s):
    c = s["case"]
    b, t, nq, nkv, hd, page = c["b"], c["t"], c["nq"], c["nkv"], c["hd"], c["page"]
    rep, rows, scale = nq // nkv, s["rows"], c["hd"] ** -0.5
    seq, place, slot = _rows(s)
    q = s["q"].float() * scale
    flat = lambda z: z.float().permute(1, 0, 2, 3).reshape(nkv, z.shape[0] * page, hd)  # noqa: E731
    pk, pv = flat(s["k"][s["prefix"].long()])[:, :c["off"]], flat(s["v"][s["prefix"].long()])[:, :c["off"]]
    qg = q.view(rows, nkv, rep, hd)
    at_prefix = qg.permute(1, 0, 2, 3).reshape(nkv, rows * rep, hd).matmul(pk.transpose(1, 2).contiguous())          # [nkv, rows * rep, off]
    own_len = s["table"].shape[1] * page
    gather = lambda z: z[s["table"].long().clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(b, nkv, own_len, hd)  # noqa: E731
    k, v = gather(s["k"]), gather(s["v"])
    padded = torch.zeros(b, nkv, t, rep, hd, device=q.device)
    padded[seq, :, place] = qg
    at_own = padded.view(b, nkv, t * rep, hd).matmul(k.transpose(2, 3).contiguous()).view(b, nkv, t, rep, own_len)[seq, :, place]   # [rows, nkv, rep, L]
    at_own = at_own.masked_fill((torch.arange(own_len, device=q.device)[None] > slot[:, None])[:, None, None], -math.inf)
    score = torch.cat((at_prefix.view(nkv, rows, rep, c["off"]).permute(1, 0, 2, 3), at_own), -1)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = p[..., :c["off"]].permute(1, 0, 2, 3).reshape(nkv, rows * rep, c["off"]).contiguous().matmul(pv.contiguous()).view(nkv, rows, rep, hd).permute(1, 0, 2, 3)
    pp = torch.zeros(b, nkv, t, rep, own_len, device=q.device)
    pp[seq, :, place] = p[..., c["off"]:]
    o = o + pp.view(b, nkv, t * rep, own_len).matmul(v).view(b, nkv, t, rep, hd)[seq, :, place]
    s["out"].copy_(torch.where((slot >= 0)[:, None, None], o.reshape(rows, nq, hd).to(s["out"].dtype), s["out"]))
    return s["out"]


def _sample_plain(s):
    x, n = s["logits"].double(), s["logits"].shape[1]
    col = lambda z: (z.double() if torch.is_tensor(z) else torch.full((x.shape[0],), float(z), dtype=torch.float64, device=x.device))[:, None]  # noqa: E731
    temp, topk, top_p, min_p = (col(s["set"][k]) for k in ("temperature", "topk", "top_p", "min_p"))
    x = torch.where(temp == 0, torch.where(x == x.amax(-1, keepdim=True), 0.0, -math.inf), x)
    w = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(temp == 0, 1.0, temp))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(n, device=x.device)[None]
    k = torch.where(temp == 0, 1.0, torch.where(topk <= 0, float(n), topk))
    keep = rank < k
    before = (ws * keep).cumsum(-1) - ws
    keep &= (before < top_p * (ws * keep).sum(-1, keepdim=True)) | (top_p >= 1)
    keep &= ws >= min_p
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter(1, order, ws * keep)
    cum = kept.cumsum(-1)
    hit = (cum > s["u"].double()[:, None] * cum[:, -1:]) & (kept > 0)
    return hit.to(torch.int32).argmax(-1, keepdim=True).to(torch.int32)


def run(s):
    c = s["case"]
    if own:
        import csm_hf_amd as csm
        if c["op"] == "append":
            csm.paged_rope_append(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["lens"], cu_rows=s["cu"], pos_offset=c["off"], q_out=s["out"])
            return s["out"], s["k"], s["v"]
        if c["op"] == "attention":
            return csm.paged_prefix_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], prefix_table=s["prefix"], prefix_len=c["off"],
                                              cu_rows=s["cu"], out=s["out"])
        return csm.sample_filtered(s["logits"], s["u"], **s["set"])
    return (_append_plain if c["op"] == "append" else _attention_plain if c["op"] == "attention" else _sample_plain)(s)


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["v"]
        return dict(bytes=n * (4 if case["x"] == "f32" else 2) + 8 * case["rows"], flops=3 * n)
    new, lens = _shape(case)
    sx, sc = (4 if case[k] == "f32" else 2 for k in ("x", "c"))
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    live = [(t, n) for t, n in zip(new, lens) if n >= 0]
    rows = sum(t for t, _ in live)
    if case["op"] == "append":
        return dict(bytes=rows * hd * ((nq + 2 * nkv) * sx + nq * sx + 2 * nkv * sc) + min(rows, case["off"] + case["own"]) * hd * 4, flops=3 * rows * (nq + nkv) * hd)
    seen = sum(t * case["off"] + t * n - t * (t - 1) // 2 for t, n in live)
    return dict(bytes=2 * rows * nq * hd * sx + (case["off"] + sum(n for _, n in live)) * 2 * nkv * hd * sc, flops=4 * seen * nq * hd)


def exact(case, seed):
    if case["op"] == "sample":
        return None
    s = prepare(case, seed)
    new, lens = _shape(case)
    nq, nkv, hd, page, off = case["nq"], case["nkv"], case["hd"], case["page"], case["off"]
    half, first = hd // 2, 0
    out, k, v = s["out"].double(), s["k"].double(), s["v"].double()
    table, prefix = s["table"].long(), s["prefix"].long()
    flat = lambda z: z.transpose(0, 1).reshape(nkv, z.shape[0] * page, hd)  # noqa: E731
    if case["op"] == "attention":
        pk, pv = flat(k[prefix])[:, :off], flat(v[prefix])[:, :off]
    for i in range(case["b"]):
        a, z, n = first, first + new[i], lens[i]
        first = z
        if n < 0:
            continue
        slots = torch.arange(n - new[i], n, device=out.device)
        if case["op"] == "append":
            x = s["qkv"][a:z].double().view(-1, nq + 2 * nkv, hd)
            ang = torch.complex(s["cos"].double(), s["sin"].double())[slots + off][:, None]
            y = torch.complex(x[:, :nq + nkv, :half], x[:, :nq + nkv, half:]) * ang
            y = torch.cat((y.real, y.imag), -1)
            out[a:z] = y[:, :nq]
            k[table[i, slots // page], :, slots % page] = y[:, nq:]
            v[table[i, slots // page], :, slots % page] = x[:, nq + nkv:]
        else:
            used = table[i, :-(-n // page)]
            ki, vi = (torch.cat((p, flat(c[used])[:, :n]), 1) for p, c in ((pk, k), (pv, v)))
            hide = torch.arange(off + n, device=out.device)[None] > off + slots[:, None]
            for h in range(nq):
                logit = (s["q"][a:z, h].double() @ ki[h // (nq // nkv)].T / math.sqrt(hd)).masked_fill(hide, -math.inf)
                out[a:z, h] = torch.softmax(logit, -1) @ vi[h // (nq // nkv)]
    return out if case["op"] == "attention" else (out, k, v)
