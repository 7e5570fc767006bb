"""Cases of the 8-bit KV cache operators: append, attention, eviction.

`listed()` names the cases, `prepare()` makes one case's inputs on the GPU,
`run()` makes one pass over them: in plain torch arithmetic (32-bit, rounded
once at the end), or, with `own` set, through tierlm_b200.kvcache. `exact()`
is the same result from the definitions in 64 bits.

The cache of one layer is a pool of pages: codes [n_pages][KV][page][hd]
(int8, or 8-bit floats e4m3) and one f32 scale per `block` rows and head,
[n_pages][KV][page / block]; row t of a sequence is row t % page of page
table[t // page]. A block holding x is stored with
d = max(max |x|, 2^-100) / Q (Q = 127 or 448) and codes round(x / d).
"""
import math

import numpy as np
import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOOR = 2.0 ** -100
DEV = "cuda"

ATTEND = dict(op="attend", fmt="int8", dtype="f32", H=32, KV=4, hd=128, page=64, block=16, n_seq=1, q=1, q_min=1,
              ctx=1024, ctx_min=1024, softcap=0.0, alibi=False, causal=True, window=0, prefix=0, docs=0, weights=False,
              evicted=False)
APPEND = dict(op="append", fmt="int8", dtype="f32", KV=4, hd=128, page=64, block=16, n_seq=1, q=1, q_min=1, ctx=1024,
              ctx_min=1024)
EVICT = dict(op="evict", fmt="int8", KV=4, hd=128, page=64, block=16, n_seq=1, ctx=1024, ctx_min=1024, keep=256,
             sink=4, recent=64)


def listed():
    return [
        # one decode step of one short conversation: launch latency is all there is
        dict(ATTEND, name="decode_bs1_701", ctx=701, ctx_min=701),
        # one decode step at the longest context: a stream of 134 MB of codes
        dict(ATTEND, name="decode_bs1_128k", ctx=131071, ctx_min=131071),
        # a serving batch of ragged conversations, capped scores, 8-bit floats, bf16 activations
        dict(ATTEND, name="decode_bs64_cap", fmt="e4m3", dtype="bf16", n_seq=64, ctx=8192, ctx_min=1, softcap=30.0),
        # a decode step that also accumulates the attention weights eviction goes by, after an earlier eviction
        dict(ATTEND, name="decode_bs16_weights", H=64, n_seq=16, ctx=4099, ctx_min=2000, alibi=True, weights=True,
             evicted=True),
        # five draft tokens per sequence checked at once, sliding window with always-visible first tokens
        dict(ATTEND, name="verify_bs24_window", dtype="bf16", H=8, KV=2, hd=64, page=16, n_seq=24, q=5, q_min=2,
             ctx=6000, ctx_min=100, window=1024, prefix=4),
        # the prompt of one request, 8-bit cache already written
        dict(ATTEND, name="prefill_2048", dtype="bf16", q=2048, q_min=2048, ctx=2048, ctx_min=2048),
        # a later chunk of a long prompt: 2,048 tokens over 18,432 rows, capped scores
        dict(ATTEND, name="prefill_chunk_18k", fmt="e4m3", dtype="bf16", page=128, block=32, q=2048, q_min=2048,
             ctx=18432, ctx_min=18432, softcap=50.0),
        # packed documents with f32 activations: every document sees only itself
        dict(ATTEND, name="prefill_docs_f32", n_seq=3, q=1500, q_min=700, ctx=1500, ctx_min=700, docs=5),
        # every sequence of a decode batch appends its token, then the rows of its block are read back
        dict(APPEND, name="append_bs64_1", n_seq=64, ctx=4096, ctx_min=16),
        # prompts of four requests appended from odd rows on, then read back
        dict(APPEND, name="append_prompt_8k", fmt="e4m3", dtype="bf16", n_seq=4, q=3001, q_min=900, ctx=3500,
             ctx_min=3020),
        # one long conversation cut to an eighth
        dict(EVICT, name="evict_32k", ctx=32768, ctx_min=32768, keep=4096, recent=512),
        # a ragged batch, some of whose sequences are short enough to stay whole
        dict(EVICT, name="evict_bs32", fmt="e4m3", block=32, n_seq=32, ctx=2047, ctx_min=100, keep=500),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: decode, a few tokens, prefill, append, evict."""
    H, KV, hd = rng.choice([(32, 4, 128), (8, 2, 64), (64, 4, 128), (16, 16, 64), (6, 2, 128), (16, 2, 256)])
    page = rng.choice([16, 32, 64, 128, 256])
    lay = dict(fmt=rng.choice(["int8", "e4m3"]), KV=KV, hd=hd, page=page, block=rng.choice([b for b in (1, 8, 16, 32, 64) if b <= page]))
    op = rng.choice(["decode", "decode", "few", "prefill", "prefill", "append", "evict"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "append":
        q = _log(rng, 1, 3000)
        n = _log(rng, 1, max(1, min(64, 8000 // q)))
        ctx = q + rng.randrange(0, 2000)
        return dict(APPEND, **lay, dtype=dtype, n_seq=n, q=q, q_min=max(1, q // 2), ctx=ctx, ctx_min=max(q, ctx // 2))
    if op == "evict":
        ctx = _log(rng, 200, 32768)
        n = _log(rng, 1, max(1, min(32, 65536 // ctx)))
        keep = max(100, int(ctx * rng.uniform(0.1, 0.7)))
        return dict(EVICT, **lay, n_seq=n, ctx=ctx, ctx_min=max(1, ctx // rng.choice([1, 2, 10])), keep=keep, recent=keep // 8)
    shape = rng.choice(["plain", "plain", "cap", "alibi", "window", "docs"])
    mods = {"plain": {}, "cap": dict(softcap=rng.choice([20.0, 30.0, 50.0])), "alibi": dict(alibi=True),
            "window": dict(window=_log(rng, 64, 4096), prefix=rng.choice([0, 4, 100])), "docs": dict(docs=rng.randrange(2, 9))}[shape]
    if op == "prefill":
        q = _log(rng, 64, 2048)
        ctx = q + rng.choice([0, rng.randrange(1, 8000)])
        n = _log(rng, 1, max(1, min(4, 3000 // q)))
        return dict(ATTEND, **lay, H=H, dtype=dtype, n_seq=n, q=q, q_min=max(1, q // 2), ctx=ctx, ctx_min=max(q, ctx // 2), **mods)
    q = 1 if op == "decode" else rng.randrange(2, 9)
    ctx = _log(rng, 100, 131071)
    n = _log(rng, 1, max(1, min(64, 262144 // ctx)))
    return dict(ATTEND, **lay, H=H, dtype=dtype, n_seq=n, q=q, q_min=1, ctx=ctx, ctx_min=max(q, ctx // rng.choice([1, 2, 50])),
                weights=rng.random() < 0.3, evicted=shape in ("plain", "alibi") and rng.random() < 0.3, **mods)


def _spread(lo, hi, n):
    """n lengths over [lo, hi], the first of them hi, without an order."""
    return [hi if s == 0 else lo + int((hi - lo) * ((0.6180339887 * s + 0.21) % 1.0)) for s in range(n)]


def _lens(c):
    L = _spread(c["ctx_min"], c["ctx"], c["n_seq"])
    if "q" not in c:
        return L, [0] * len(L)
    return L, [min(a, b) for a, b in zip(L, _spread(c["q_min"], c["q"], c["n_seq"])[::-1])]


def _doc_cuts(c, n):
    """First positions of the documents that fill positions [0, n)."""
    return sorted({0} | {1 + int((n - 1) * ((0.7548776662 * i + 0.1) % 1.0)) for i in range(1, c["docs"])})


def _pairs(c, n, q):
    """(query, key) pairs that the masks leave of a sequence of n rows, q of them queries, and the rows read."""
    pos = np.arange(n - q, n)
    first = np.zeros_like(pos)
    if c["docs"]:
        cuts = np.array(_doc_cuts(c, n))
        first = cuts[np.searchsorted(cuts, pos, side="right") - 1]
    if c["window"]:
        first = np.maximum(first, pos - c["window"] + 1)
    seen = pos - first + 1
    pre = np.minimum(first, c["prefix"]) if c["window"] and not c["docs"] else 0
    return int((seen + pre).sum()), int(min(n, n - first.min() + np.max(pre)))


def work(case):
    c = case
    L, Q = _lens(c)
    KV, hd = c["KV"], c["hd"]
    row = 2 * KV * (hd + 4.0 / c["block"])
    if c["op"] == "append":
        es = 2 if c["dtype"] == "bf16" else 4
        n = sum(Q)
        back = sum(l - (l - q) // c["block"] * c["block"] for l, q in zip(L, Q))
        old = back - n
        # the new rows in, their codes and scales out; the old rows of a begun block in and out; the rows read back as f32
        return {"bytes": n * 2 * KV * hd * es + n * row + 2 * old * row + back * (row + 2 * KV * hd * 4), "flops": 4 * n * KV * hd}
    if c["op"] == "evict":
        kept = sum(min(l, c["keep"]) for l in L)
        # every weight in; the kept rows in and out with their weights, indices and positions, then read back as f32
        return {"bytes": sum(L) * KV * 4 + kept * (2 * row + KV * 16) + kept * (row + 2 * KV * hd * 4), "flops": 4 * kept * KV * hd}
    H, es = c["H"], 2 if c["dtype"] == "bf16" else 4
    got = [_pairs(c, l, q) for l, q in zip(L, Q)]
    pairs, rows = sum(p for p, _ in got), sum(r for _, r in got)
    extra = rows * KV * 4 * ((1 if c["evicted"] else 0) + (2 if c["weights"] else 0))
    return {"bytes": rows * row + sum(Q) * H * (2 * hd * es + 4) + extra, "flops": 4.0 * hd * H * pairs}


# ---- inputs ------------------------------------------------------------------
def _store(x, fmt, block):
    """x f32 [..., rows, hd] -> codes and scales [..., rows / block] (rows a multiple of block)."""
    y = x.unflatten(-2, (-1, block))
    d = y.abs().amax((-1, -2)).clamp_min(FLOOR) / QMAX[fmt]
    y = y / d[..., None, None]
    y = y.round() if fmt == "int8" else y.clamp(-448, 448)
    return y.to(CODE[fmt]).flatten(-3, -2), d


def _pools(c, g, n_pages):
    """K and V pools full of rows as a model writes them: K with a few large channels, V plain."""
    shape = (n_pages, c["KV"], c["page"], c["hd"])
    chan = 1 + 2 * (torch.rand((c["KV"], 1, c["hd"]), generator=g, device=DEV) > 0.95)
    out = {}
    for name in ("k", "v"):
        codes = torch.empty(shape, dtype=CODE[c["fmt"]], device=DEV)
        scale = torch.empty((n_pages, c["KV"], c["page"] // c["block"]), device=DEV)
        step = max(1, (1 << 26) // (c["KV"] * c["page"] * c["hd"]))
        for p in range(0, n_pages, step):
            x = torch.randn((min(step, n_pages - p), *shape[1:]), generator=g, device=DEV)
            codes[p:p + step], scale[p:p + step] = _store(x * chan if name == "k" else x, c["fmt"], c["block"])
        out[name], out[name + "_scale"] = codes, scale
    return out


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(g, lens, page, n_pages, stride):
    """A page table [n_seq][stride] over shuffled pages; entries past a sequence's end are 0."""
    perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    need = _int([-(-l // page) for l in lens])
    at = torch.arange(stride, device=DEV)[None, :]
    base = (need.cumsum(0) - need)[:, None]
    return torch.where(at < need[:, None], perm[(base + at).clamp_max(n_pages - 1).long()], 0).to(torch.int32).contiguous()


def _starts(n):
    return [0] + list(np.cumsum(n))


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    L, Q = _lens(c)
    page = c["page"]
    stride = -(-max(L) // page)
    n_used = sum(-(-l // page) for l in L)
    st = {"case": c, "max_kv": max(L), "max_q": max(max(Q), 1), "kv_len": _int(L), "q_start": _int(_starts(Q)),
          "lens": L, "q_lens": Q}
    st["table"] = _table(g, L, page, n_used, stride)
    if c["op"] == "evict":
        kept = [min(l, c["keep"]) for l in L]
        n_dst = sum(-(-l // page) for l in kept)
        st.update(_pools(c, g, n_used + n_dst))
        # the pages of the kept rows are other pages of the same pool
        perm = _table(g, kept, page, n_dst, -(-max(kept) // page))
        st["dst_table"] = torch.where(torch.arange(perm.shape[1], device=DEV)[None] < (_int([-(-l // page) for l in kept]))[:, None], perm + n_used, 0).to(torch.int32).contiguous()
        st["pos"] = torch.arange(page, device=DEV, dtype=torch.int32).expand(n_used + n_dst, c["KV"], page).contiguous()
        stride_w = max(L)
        # accumulated weights: a heavy tail, many equal small ones, as rounding leaves them
        w = torch.rand((c["n_seq"], c["KV"], stride_w), generator=g, device=DEV).pow(6) * 50
        st["weights"] = torch.where(w < 0.02, torch.full_like(w, 0.01), w)
        st["weights_out"] = torch.zeros((c["n_seq"], c["KV"], c["keep"]), device=DEV)
        st["read_row0"], st["read_start"], st["read_total"] = _int([0] * len(L)), _int(_starts(kept)), sum(kept)
        st["kept"] = kept
    else:
        st.update(_pools(c, g, n_used))
        dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
        total = sum(Q)
        if c["op"] == "append":
            st["new_k"] = (torch.randn((total, c["KV"], c["hd"]), generator=g, device=DEV) * 1.5).to(dt)
            st["new_v"] = torch.randn((total, c["KV"], c["hd"]), generator=g, device=DEV).to(dt)
            row0 = [(l - q) // c["block"] * c["block"] for l, q in zip(L, Q)]
            back = [l - r for l, r in zip(L, row0)]
            st["read_row0"], st["read_start"], st["read_total"] = _int(row0), _int(_starts(back)), sum(back)
            st["back"] = back
        else:
            st["query"] = (torch.randn((total, c["H"], c["hd"]), generator=g, device=DEV) * 1.5).to(dt)
            st["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["H"] + 1, device=DEV) / c["H"]) if c["alibi"] else None
            st["prefix"] = _int([c["prefix"]] * c["n_seq"]) if c["prefix"] else None
            st["doc"] = st["pos"] = st["q_pos"] = st["acc"] = None
            if c["docs"]:
                doc = np.full((c["n_seq"], max(L)), -1, np.int32)
                for s, l in enumerate(L):
                    doc[s, :l] = np.searchsorted(np.array(_doc_cuts(c, l)), np.arange(l), side="right") - 1
                st["doc"] = torch.from_numpy(doc).to(DEV)
            if c["evicted"]:
                # rows kept of a sequence three times as long, other ones for each head
                gap = torch.randint(1, 6, (c["n_seq"], c["KV"], max(L)), generator=g, device=DEV, dtype=torch.int32)
                rows = gap.cumsum(2).to(torch.int32)
                st["pos"] = torch.zeros((n_used, c["KV"], page), dtype=torch.int32, device=DEV)
                s, t = _rows(st)
                p = st["table"][s, t // page].long()
                st["pos"][p, :, t % page] = rows[s, :, t]
                s, t = _queries(st)
                st["q_pos"] = (rows[s, :, t].amax(1)).to(torch.int32)
            if c["weights"]:
                st["acc"] = torch.zeros((c["n_seq"], c["KV"], max(L)), device=DEV)
    if own:
        from tierlm_b200 import kvcache as K
        st["cache"] = K.Kv8Cache.from_pools(st["k"], st["v"], st["k_scale"], st["v_scale"], st.get("pos"))
        st["batch"] = K.Kv8Batch(st["table"], st["q_start"], st["kv_len"], st["max_q"], st["max_kv"], st.get("q_pos"))
        if c["op"] == "attend":
            st["score"] = K.Score(softcap=c["softcap"], slopes=st["slopes"], causal=c["causal"], window=c["window"], prefix=st["prefix"], doc=st["doc"])
    return st


def _rows(st):
    """(sequence, row) of every row that the cache holds."""
    s = torch.repeat_interleave(torch.arange(len(st["lens"]), device=DEV), st["kv_len"].long(), output_size=sum(st["lens"]))
    first = st["kv_len"].long().cumsum(0) - st["kv_len"].long()
    return s, torch.arange(s.numel(), device=DEV) - first[s]


def _queries(st):
    """(sequence, row) of every new token."""
    n = st["q_start"][1:].long() - st["q_start"][:-1].long()
    s = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=sum(st["q_lens"]))
    return s, torch.arange(s.numel(), device=DEV) - st["q_start"].long()[s] + (st["kv_len"].long() - n)[s]


# ---- one pass ----------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "evict": _own_evict}[c["op"]](state)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[c["op"]](state)


def _own_append(st):
    cache = st["cache"]
    cache.append(st["new_k"], st["new_v"], st["batch"])
    k, v = cache.read(st["table"], st["read_row0"], st["read_start"], st["read_total"])
    return {"k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}


def _own_attend(st):
    out, lse = st["cache"].attend(st["query"], st["batch"], st["score"], weights=st["acc"], lse=True)
    r = {"out": out, "lse": lse}
    if st["acc"] is not None:
        r["weights"] = st["acc"]
    return r


def _own_evict(st):
    c, cache = st["case"], st["cache"]
    rows, lens = cache.evict(st["weights"], st["batch"], st["dst_table"], c["keep"], sink=c["sink"], recent=c["recent"], weights_out=st["weights_out"])
    k, v = cache.read(st["dst_table"], st["read_row0"], st["read_start"], st["read_total"])
    return {"rows": rows, "lens": lens, "k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale, "pos": cache.pos, "weights": st["weights_out"]}


def _values(st, name, s, t, table="table"):
    """The f32 values [n][KV][hd] of rows t of sequences s."""
    c = st["case"]
    p, r = st[table][s, t // c["page"]].long(), t % c["page"]
    return st[name][p, :, r].float() * st[name + "_scale"][p, :, r // c["block"]][..., None]


def _put(st, name, s, t, codes, table="table"):
    p, r = st[table][s, t // st["case"]["page"]].long(), t % st["case"]["page"]
    st[name].view(torch.uint8)[p, :, r] = codes.view(torch.uint8)


def _round(y, fmt):
    return (y.round() if fmt == "int8" else y.clamp(-448, 448)).to(CODE[fmt])


def _read_rows(st):
    n = st["read_start"][1:].long() - st["read_start"][:-1].long()
    s = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=st["read_total"])
    return s, torch.arange(s.numel(), device=DEV) - st["read_start"].long()[s] + st["read_row0"].long()[s]


def _plain_append(st):
    c = st["case"]
    s, t = _read_rows(st)                       # every row of a touched block, the new ones last
    n_new = st["q_start"][1:].long() - st["q_start"][:-1].long()
    first = (st["kv_len"].long() - n_new)[s]
    new = t >= first
    src = (t - first + st["q_start"].long()[s]).clamp_min(0)
    blk = s * (-(-st["max_kv"] // c["block"])) + t // c["block"]
    n_blk = c["n_seq"] * (-(-st["max_kv"] // c["block"]))
    p, b = st["table"][s, t // c["page"]].long(), t % c["page"] // c["block"]
    begun = t // c["block"] * c["block"] < first     # the block has rows of earlier calls
    res = {}
    for name in ("k", "v"):
        x = torch.where(new[:, None, None], st["new_" + name][src].float(), _values(st, name, s, t))
        top = torch.where(new[:, None], x.abs().amax(2), 0)
        top = torch.zeros((n_blk, c["KV"]), device=DEV).index_reduce_(0, blk, top, "amax")
        d = (top.clamp_min(FLOOR) / QMAX[c["fmt"]])[blk]
        d = torch.where(begun[:, None], torch.maximum(d, st[name + "_scale"][p, :, b]), d)
        codes = _round(x / d[..., None], c["fmt"])
        _put(st, name, s, t, codes)
        st[name + "_scale"][p, :, b] = d
        res[name] = _values(st, name, s, t)
    return {"k": res["k"], "v": res["v"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _plain_attend(st):
    c = st["case"]
    n_seq, KV, H, hd, T = c["n_seq"], c["KV"], c["H"], c["hd"], st["max_kv"]
    n, G = st["max_q"], H // KV
    # the cache as f32 [n_seq][KV][T][hd]; rows past a sequence's end are masked below
    t = torch.arange(T, device=DEV)
    page = st["table"].long()[:, t // c["page"]]
    keys = {name: (st[name][page, :, t % c["page"]].float() * st[name + "_scale"][page, :, t % c["page"] // c["block"]][..., None]).transpose(1, 2) for name in ("k", "v")}
    s_id, row = _queries(st)
    slot = torch.arange(s_id.numel(), device=DEV) - st["q_start"].long()[s_id]
    q = torch.zeros((n_seq, n, H, hd), device=DEV)
    q[s_id, slot] = st["query"].float()
    q = q.view(n_seq, n, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, KV, G * n, hd)
    q_row = torch.zeros((n_seq, n), dtype=torch.long, device=DEV)
    q_row[s_id, slot] = row
    if st["q_pos"] is not None:
        q_at = torch.zeros((n_seq, n), dtype=torch.long, device=DEV)
        q_at[s_id, slot] = st["q_pos"].long()
        k_at = st["pos"][page, :, t % c["page"]].transpose(1, 2).long()
    else:
        q_at, k_at = q_row, t.expand(n_seq, KV, T)
    far = q_at[:, None, :, None] - k_at[:, :, None, :]                       # [n_seq][KV][n][T]
    seen = (t[None] < st["kv_len"][:, None])[:, None, None, :] & torch.ones_like(far, dtype=torch.bool)
    near = torch.ones_like(seen)
    if c["causal"]:
        near = near & (far >= 0)
    if c["window"]:
        near = near & (far < c["window"])
    if st["prefix"] is not None:
        near = near | (k_at < st["prefix"].long()[:, None, None])[:, :, None, :]
    seen = seen & near
    if st["doc"] is not None:
        dq = st["doc"].gather(1, q_at)
        seen = seen & (dq[:, None, :, None] == st["doc"][:, None, None, :T])
    z = torch.matmul(q, keys["k"].transpose(2, 3)) * (1.0 / math.sqrt(hd))
    if c["softcap"]:
        z = c["softcap"] * torch.tanh(z / c["softcap"])
    z = z.view(n_seq, KV, G, n, T)
    if st["slopes"] is not None:
        z = z - st["slopes"].view(KV, G)[None, :, :, None, None] * far.abs()[:, :, None].float()
    z = z.masked_fill(~seen[:, :, None], float("-inf"))
    top = z.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    z = torch.exp(z - top)
    total = z.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    z = z / torch.where(total == 0, 1.0, total)
    out = torch.matmul(z.view(n_seq, KV, G * n, T), keys["v"]).view(n_seq, KV, G, n, hd)
    out = out.permute(0, 3, 1, 2, 4).reshape(n_seq, n, H, hd)[s_id, slot]
    lse = lse[..., 0].permute(0, 3, 1, 2).reshape(n_seq, n, H)[s_id, slot]
    r = {"out": out.to(st["query"].dtype), "lse": lse}
    if st["acc"] is not None:
        real = torch.arange(n, device=DEV)[None] < (st["q_start"][1:] - st["q_start"][:-1])[:, None]
        st["acc"] += (z * real[:, None, None, :, None]).sum((2, 3))
        r["weights"] = st["acc"]
    return r


def _plain_evict(st):
    c = st["case"]
    n_seq, KV, keep, T = c["n_seq"], c["KV"], c["keep"], st["max_kv"]
    t = torch.arange(T, device=DEV)
    L = st["kv_len"].long()[:, None, None]
    w = st["weights"].masked_fill((t < c["sink"]) | (t >= L - c["recent"]), float("inf")).masked_fill(t >= L, float("-inf"))
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(torch.arange(order.shape[-1], device=DEV) < L, order, T)
    order = torch.sort(order, dim=-1).values
    order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=T)
    rows = torch.where(order < T, order, -1).to(torch.int32)
    lens = st["kv_len"].clamp_max(keep)
    s, j = _read_rows(st)                                   # kept rows: sequence, place
    head = torch.arange(KV, device=DEV)[None]
    src = rows[s, :, j].long()                              # [n][KV]
    p, r = st["table"].long()[s[:, None], src // c["page"]], src % c["page"]
    dp, dr = st["dst_table"][s, j // c["page"]].long(), j % c["page"]
    nb = -(-keep // c["block"])
    blk = s * nb + j // c["block"]
    res = {}
    for name in ("k", "v"):
        x = st[name][p, head, r].float() * st[name + "_scale"][p, head, r // c["block"]][..., None]
        top = torch.zeros((n_seq * nb, KV), device=DEV).index_reduce_(0, blk, x.abs().amax(2), "amax")
        d = (top.clamp_min(FLOOR) / QMAX[c["fmt"]])[blk]
        _put(st, name, s, j, _round(x / d[..., None], c["fmt"]), "dst_table")
        st[name + "_scale"][dp, :, dr // c["block"]] = d
        res[name] = _values(st, name, s, j, "dst_table")
    st["pos"][dp, :, dr] = st["pos"][p, head, r]
    got = torch.gather(st["weights"], 2, rows.clamp_min(0).long())
    st["weights_out"].copy_(torch.where(rows < 0, 0.0, got))
    return {"rows": rows, "lens": lens, "k": res["k"], "v": res["v"], "k_scale": st["k_scale"], "v_scale": st["v_scale"], "pos": st["pos"], "weights": st["weights_out"]}


# ---- the definitions in 64 bits ------------------------------------------------
def _seq_values(st, name, s, n, table="table"):
    """Rows 0..n-1 of sequence s in f64, [n][KV][hd]."""
    c = st["case"]
    pages = st[table][s, :-(-n // c["page"])].long()
    x = st[name][pages].double() if c["fmt"] == "int8" else st[name][pages].float().double()
    x = x * st[name + "_scale"][pages].double().repeat_interleave(c["block"], 2)[..., None]
    return x.transpose(1, 2).flatten(0, 1)[:n]


def _quantised(x, fmt, block, old=None):
    """x f64 [rows][KV][hd], rows from a block's begin on -> the values its codes stand for and the scales [blocks][KV].

    old = (n, d): the first n rows were there before, in a block of scale d [KV]."""
    n = x.shape[0]
    nb = -(-n // block)
    top = torch.zeros((nb * block, x.shape[1]), dtype=torch.float64, device=DEV)
    top[:n] = x.abs().amax(2)
    if old is not None:
        top[:old[0]] = 0
    d = top.view(nb, block, -1).amax(1).clamp_min(FLOOR) / QMAX[fmt]
    if old is not None and old[0]:
        d[0] = torch.maximum(d[0], old[1])
    r = d.repeat_interleave(block, 0)[:n, :, None]
    y = x / r
    y = torch.round(y) if fmt == "int8" else y.float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
    return y * r, d


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[c["op"]](st, c)


def _exact_append(st, c):
    res = {"k": [], "v": []}
    for name in ("k", "v"):
        scale = st[name + "_scale"].double()
        for s, (l, q, back) in enumerate(zip(st["lens"], st["q_lens"], st["back"])):
            row0, at = l - back, sum(st["q_lens"][:s])
            x = _seq_values(st, name, s, l)[row0:].clone()
            x[back - q:] = st["new_" + name][at:at + q].double()
            blocks = torch.arange(row0 // c["block"], -(-l // c["block"]), device=DEV)
            per = c["page"] // c["block"]
            p, b = st["table"][s].long()[blocks // per], blocks % per
            y, d = _quantised(x, c["fmt"], c["block"], (back - q, scale[p[0], :, b[0]]))
            scale[p, :, b] = d
            res[name].append(y)
        res[name + "_scale"] = scale
    return {"k": torch.cat(res["k"]), "v": torch.cat(res["v"]), "k_scale": res["k_scale"], "v_scale": res["v_scale"]}


def _exact_attend(st, c):
    outs, lses = [], []
    acc = None if st["acc"] is None else st["acc"].double().clone()
    G = c["H"] // c["KV"]
    for s, (l, q) in enumerate(zip(st["lens"], st["q_lens"])):
        at = sum(st["q_lens"][:s])
        k, v = _seq_values(st, "k", s, l), _seq_values(st, "v", s, l)
        x = st["query"][at:at + q].double()
        out = torch.empty((q, c["H"], c["hd"]), dtype=torch.float64, device=DEV)
        lse = torch.empty((q, c["H"]), dtype=torch.float64, device=DEV)
        qp = (torch.arange(l - q, l, device=DEV) if st["q_pos"] is None else st["q_pos"][at:at + q].long())[:, None]
        for h in range(c["H"]):
            kv = h // G
            if st["pos"] is None:
                kp = torch.arange(l, device=DEV)[None]
            else:
                kp = st["pos"][st["table"][s, :-(-l // c["page"])].long(), kv].flatten()[:l].long()[None]
            ok = kp <= qp
            if c["window"]:
                ok = ok & (qp - kp < c["window"])
            if c["prefix"]:
                ok = ok | (kp < c["prefix"])
            if st["doc"] is not None:
                ok = ok & (st["doc"][s][kp] == st["doc"][s][qp])
            z = x[:, h] @ k[:, kv].T / math.sqrt(c["hd"])
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            if c["alibi"]:
                z = z - st["slopes"][h].double() * (qp - kp).abs()
            z = torch.where(ok, z, -math.inf)
            lse[:, h] = torch.logsumexp(z, 1)
            p = torch.nan_to_num(torch.exp(z - lse[:, h, None]), nan=0.0)
            out[:, h] = p @ v[:, kv]
            if acc is not None:
                acc[s, kv, :l] += p.sum(0)
        outs.append(out)
        lses.append(lse)
    r = {"out": torch.cat(outs), "lse": torch.cat(lses)}
    if acc is not None:
        r["weights"] = acc
    return r


def _exact_evict(st, c):
    res = {"k": [], "v": []}
    w = st["weights"].double().cpu().numpy()
    kept = [[None] * c["KV"] for _ in st["lens"]]
    w_out = np.zeros((c["n_seq"], c["KV"], c["keep"]))
    for s, l in enumerate(st["lens"]):
        n = min(l, c["keep"])
        for h in range(c["KV"]):
            t = np.arange(l)
            held = (t < c["sink"]) | (t >= l - c["recent"])
            order = np.lexsort((t, -w[s, h, :l], ~held))[:n]
            kept[s][h] = np.sort(order)
            w_out[s, h, :n] = w[s, h, kept[s][h]]
    per = c["page"] // c["block"]
    for name in ("k", "v"):
        scale = st[name + "_scale"].double()
        for s, l in enumerate(st["lens"]):
            n = st["kept"][s]
            x = _seq_values(st, name, s, l)
            x = torch.stack([x[torch.from_numpy(kept[s][h]).to(DEV), h] for h in range(c["KV"])], 1)
            y, d = _quantised(x, c["fmt"], c["block"])
            blocks = torch.arange(d.shape[0], device=DEV)
            scale[st["dst_table"][s].long()[blocks // per], :, blocks % per] = d
            res[name].append(y)
        res[name + "_scale"] = scale
    return {"rows": None, "lens": None, "k": torch.cat(res["k"]), "v": torch.cat(res["v"]), "k_scale": res["k_scale"], "v_scale": res["v_scale"], "pos": None,
            "weights": torch.from_numpy(w_out).to(DEV)}
