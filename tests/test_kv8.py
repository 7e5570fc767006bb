"""The 8-bit KV cache (tierlm_b200/kvcache.py): append, read-back, attention,
selection and compaction.

CPU: the C calls' refusals (they are checked before any GPU call) and the
wrapper's. GPU: codes, scales, positions and kept rows equal a NumPy
restatement bit for bit; attention against a 64-bit one.

Attention tolerances. Let A = max over a query's visible keys of scale *
sum |q_i k_i|. A score is off by at most ds = A * 2^-19 + 2^-20 * (|softcap| +
|slope * distance|): the query's two f16 parts keep 22 bits, the tensor
core adds hd / 16 <= 16 products of 16 terms with truncation (2^-23 each, of
at most A), three roundings follow (2^-24 each). A softmax weight is then off by
a factor within 1 +- (2 ds + 2^-18), the sums of up to 2^14 positive terms taken
in pieces of 8 and joined included, so |out - ref| <= (2 ds + 2^-18) sum
p |v|, plus 2^-11 sum p |v| where probabilities enter as one f16, plus half of
f16's smallest step, 2^-39 of the largest product of p and a row's scale per unit
of |code| (2^-50 for f32 queries, whose remainders are carried times 2^11), plus
the output's own rounding (2^-8 of it for bf16, 2^-11 for f16). lse is off by ds +
2^-18 + 2^-22 |lse|, an accumulated weight by its factor.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

from tierlm_b200 import TlmError, _lib
from tierlm_b200 import kvcache as K

FLOOR = np.float32(2.0 ** -100)
INV_Q = {K.INT8: np.float32(1) / np.float32(127), K.E4M3: np.float32(1) / np.float32(448)}
CODE = {K.INT8: torch.int8, K.E4M3: torch.float8_e4m3fn}


# ---- restatement ---------------------------------------------------------------
def code_values(codes: np.ndarray, fmt: int) -> np.ndarray:
    """uint8 codes -> f32 values before the scale."""
    t = torch.from_numpy(np.ascontiguousarray(codes).view(np.uint8))
    return t.view(CODE[fmt]).float().numpy()


def to_codes(y: np.ndarray, fmt: int) -> np.ndarray:
    y = np.asarray(y, np.float32)
    if fmt == K.INT8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    return torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def quantise(x: np.ndarray, fmt: int, d=None) -> tuple[np.ndarray, np.float32]:
    """One block [rows][hd] f32 -> codes, scale."""
    if d is None:
        d = block_scale(x, fmt)
    if np.isnan(d):
        return np.zeros(x.shape, np.uint8), d
    return to_codes(x / d, fmt), d


def block_scale(x: np.ndarray, fmt: int) -> np.float32:
    if x.size == 0:
        return FLOOR * INV_Q[fmt]
    if not np.isfinite(x).all():
        return np.float32(np.nan)
    return np.maximum(np.abs(x).max().astype(np.float32), FLOOR) * INV_Q[fmt]


class Host:
    """A cache on the host: uint8 codes, f32 scales, positions."""

    def __init__(self, n_pages, KV, page, hd, fmt, block, pos=False, seed=0):
        r = np.random.default_rng(seed)
        # unwritten rows hold anything, NaN patterns among it
        self.k = r.integers(0, 256, (n_pages, KV, page, hd)).astype(np.uint8)
        self.v = r.integers(0, 256, (n_pages, KV, page, hd)).astype(np.uint8)
        self.ks = np.full((n_pages, KV, page // block), np.nan, np.float32)
        self.vs = np.full((n_pages, KV, page // block), np.nan, np.float32)
        self.pos = r.integers(0, 1 << 30, (n_pages, KV, page)).astype(np.int32) if pos else None
        self.page, self.block, self.fmt, self.KV, self.hd = page, block, fmt, KV, hd

    def gpu(self):
        dt = CODE[self.fmt]
        up = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        return K.Kv8Cache.from_pools(up(self.k).view(dt), up(self.v).view(dt), up(self.ks), up(self.vs),
                                     None if self.pos is None else up(self.pos))

    def append(self, k, v, table, q_start, kv_len, q_pos=None):
        """k, v f32 [n][KV][hd]."""
        for s in range(len(kv_len)):
            n = q_start[s + 1] - q_start[s]
            first, L = kv_len[s] - n, kv_len[s]
            if n == 0:
                continue
            for b in range(first // self.block, -(-L // self.block)):
                t0, t1 = b * self.block, min(L, (b + 1) * self.block)
                ta = max(t0, first)
                e, r = table[s, t0 // self.page], t0 % self.page
                for h in range(self.KV):
                    for x, codes, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                        new = x[q_start[s] + ta - first:q_start[s] + t1 - first, h]
                        d = block_scale(new, self.fmt)
                        if t0 < ta:
                            old = scale[e, h, r // self.block]
                            d = np.maximum(d, old)      # NaN stays
                            rows = code_values(codes[e, h, r:r + ta - t0], self.fmt) * old
                            if not d == old:
                                codes[e, h, r:r + ta - t0] = quantise(rows, self.fmt, d)[0]
                        codes[e, h, r + ta - t0:r + t1 - t0] = quantise(new, self.fmt, d)[0]
                        scale[e, h, r // self.block] = d
                    if self.pos is not None:
                        for t in range(ta, t1):
                            self.pos[e, h, r + t - t0] = t if q_pos is None else q_pos[q_start[s] + t - first]

    def rows(self, which, table_row, n):
        """Rows 0..n-1 [n][KV][hd] f64, and per row [n][KV] positions."""
        codes, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        out = np.empty((n, self.KV, self.hd))
        for t in range(n):
            e, r = table_row[t // self.page], t % self.page
            with np.errstate(invalid="ignore"):
                out[t] = code_values(codes[e, :, r], self.fmt).astype(np.float64) * scale[e, :, r // self.block][:, None].astype(np.float64)
        return out

    def scales(self, table_row, n):
        t = np.arange(n)
        return self.vs[table_row[t // self.page], :, t % self.page // self.block].astype(np.float64)

    def positions(self, table_row, n):
        t = np.arange(n)
        if self.pos is None:
            return np.repeat(t[:, None], self.KV, 1)
        return self.pos[table_row[t // self.page], :, t % self.page]


def tables(rng, lens, page, spare=2):
    need = [max(1, -(-n // page)) for n in lens]
    perm = rng.permutation(sum(need) + spare)
    t = np.full((len(lens), max(need)), -7, np.int32)    # entries past the end are never followed
    o = 0
    for s, n in enumerate(need):
        t[s, :n] = perm[o:o + n]
        o += n
    return t, sum(need) + spare


def up(a, dtype=None):
    if a is None:
        return None
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def reference(host, q, table, q_start, kv_len, H, scale=0.0, softcap=0.0, slopes=None, causal=True, window=0, prefix=None,
              doc=None, q_pos=None):
    """64-bit attention: out, lse, weights [s][KV][max L], and the bounds' terms: ds [n][H], (sum p|v|, f16 floor) [n][H][hd]."""
    G = H // host.KV
    n_all = q.shape[0]
    out, mag, low = (np.zeros((n_all, H, host.hd)) for _ in range(3))
    lse, ds = np.full((n_all, H), -np.inf), np.zeros((n_all, H))
    w = np.zeros((len(kv_len), host.KV, max(kv_len)))
    w_err = np.zeros_like(w)
    sc = scale or 1 / math.sqrt(host.hd)
    for s, L in enumerate(kv_len):
        n = q_start[s + 1] - q_start[s]
        k, v = host.rows("k", table[s], L), host.rows("v", table[s], L)
        vs = host.scales(table[s], L)
        pos = host.positions(table[s], L)
        for i in range(n):
            a = q_start[s] + i
            qp = L - n + i if q_pos is None else int(q_pos[a])
            for h in range(H):
                kv = h // G
                kp = pos[:, kv].astype(np.int64)
                see = np.ones(L, bool)
                if causal:
                    see &= kp <= qp
                if window:
                    see &= qp - kp < window
                if prefix is not None:
                    see |= kp < prefix[s]
                if doc is not None:
                    at = lambda p: np.where((p >= 0) & (p < doc.shape[1]), doc[s][np.clip(p, 0, doc.shape[1] - 1)], -1)  # noqa: E731
                    see &= at(kp) == at(np.int64(qp))
                idx = np.nonzero(see)[0]
                if idx.size == 0:
                    continue
                kk, x = k[idx, kv], q[a, h].astype(np.float64)
                z = sc * (kk @ x)
                e = 2.0 ** -19 * sc * (np.abs(kk) @ np.abs(x)).max()
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                    e += 2.0 ** -20 * softcap
                if slopes is not None:
                    far = np.abs(qp - kp[idx])
                    z = z - float(slopes[h]) * far
                    e += 2.0 ** -20 * float(slopes[h]) * far.max()
                m = z.max()
                p = np.exp(z - m)
                lse[a, h], ds[a, h] = m + math.log(p.sum()), e
                p /= p.sum()
                low[a, h] = 2.0 ** -39 * (p * vs[idx, kv]).max() * (np.abs(v[idx, kv]) / vs[idx, kv, None]).sum(0)
                out[a, h], mag[a, h] = p @ v[idx, kv], p @ np.abs(v[idx, kv])
                w[s, kv, idx] += p
                w_err[s, kv, idx] += p * (2 * e + 2.0 ** -18)
    return out, lse, w, ds, (mag, low), w_err


def assert_close(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert (np.isnan(got) == np.isnan(want)).all(), what
    ok = np.isfinite(want)
    assert (got[~ok & ~np.isnan(want)] == want[~ok & ~np.isnan(want)]).all(), what
    bad = np.abs(got - want)[ok] > np.broadcast_to(bound, want.shape)[ok]
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - want)[ok].max()))


def out_bound(want, mags, ds, dtype):
    mag, low = mags
    b = (2 * ds[..., None] + 2.0 ** -18) * mag + 2.0 ** -11 * low + 1e-37
    if dtype != torch.float32:
        b = b + 2.0 ** -11 * mag + low
        b = b * 1.01 + np.abs(want) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11) + (2.0 ** -24 if dtype == torch.float16 else 0)
    return b


def make(seed, lens, news, H, KV, hd, fmt=K.INT8, page=16, block=16, pos=False, q_scale=1.5, spread=1.0, dtype=torch.float32):
    """A filled host cache, its batch arrays and queries (rounded to dtype)."""
    rng = np.random.default_rng(seed)
    table, n_pages = tables(rng, lens, page)
    host = Host(n_pages, KV, page, hd, fmt, block, pos, seed)
    start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(start[-1])
    mult = np.exp(rng.normal(0, spread, (n, KV, 1))) if spread else 1.0
    k = (rng.standard_normal((n, KV, hd)) * mult).astype(np.float32)
    v = (rng.standard_normal((n, KV, hd)) * mult).astype(np.float32)
    host.append(k, v, table, start, lens)
    q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    q = torch.from_numpy((rng.standard_normal((int(q_start[-1]), H, hd)) * q_scale).astype(np.float32)).to(dtype)
    return host, table, q_start, q, rng


def batch(table, q_start, lens, q_pos=None, max_q=None, max_kv=None):
    n = np.diff(q_start)
    return K.Kv8Batch(up(np.asarray(table, np.int32)), up(np.asarray(q_start, np.int32)), up(np.asarray(lens, np.int32)),
                      int(n.max()) if max_q is None else max_q, int(max(lens)) if max_kv is None else max_kv,
                      up(None if q_pos is None else np.asarray(q_pos, np.int32)))


def check_attend(host, table, q_start, lens, q, H, q_pos=None, weights=False, max_kv=None, **mods):
    ref_mods = dict(mods)
    score = K.Score(scale=mods.get("scale", 0.0), softcap=mods.get("softcap", 0.0), slopes=up(mods.get("slopes")),
                    causal=mods.get("causal", True), window=mods.get("window", 0), prefix=up(mods.get("prefix")),
                    doc=up(mods.get("doc")))
    cache = host.gpu()
    b = batch(table, q_start, lens, q_pos, max_kv=max_kv)
    w = torch.full((len(lens), host.KV, max(lens) + 3), 0.5, device="cuda") if weights else None
    out, lse = cache.attend(q.cuda(), b, score, lse=True, weights=w)
    want, wlse, ww, ds, mag, w_err = reference(host, q.float().numpy(), table, q_start, lens, H, q_pos=q_pos, **ref_mods)
    assert out.dtype == q.dtype
    assert_close(out.float().cpu().numpy(), want, out_bound(want, mag, ds, q.dtype), "out")
    with np.errstate(invalid="ignore"):
        assert_close(lse.cpu().numpy(), wlse, ds + 2.0 ** -18 + 2.0 ** -22 * np.abs(np.where(np.isfinite(wlse), wlse, 0)), "lse")
    if weights:
        got = w.cpu().numpy()
        assert (got[..., max(lens):] == 0.5).all()
        for s, L in enumerate(lens):
            assert (got[s, :, L:] == 0.5).all()
        assert_close(got[..., :max(lens)] - 0.5, ww, w_err + 2.0 ** -22, "weights")   # the sum is rounded at 0.5
    return out, lse


# ---- refusals (no GPU) ------------------------------------------------------------
def c_cache(**kw):
    f = dict(k=1 << 20, v=1 << 21, k_scale=1 << 22, v_scale=1 << 23, pos=1 << 24, fmt=1, n_pages=8, KV=2, page=16, block=16, hd=64)
    f.update(kw)
    return K._Cache(**f)


def c_batch(**kw):
    f = dict(page_table=1 << 20, q_start=1 << 21, kv_len=1 << 22, q_pos=None, n_seq=2, table_stride=4, total_q=2, max_q=1, max_kv=40)
    f.update(kw)
    return K._Batch(**f)


def c_score(**kw):
    f = dict(scale=0.0, softcap=0.0, slopes=None, prefix=None, doc=None, doc_stride=0, causal=1, window=0)
    f.update(kw)
    return K._Score(**f)


BAD_CACHES = [(dict(fmt=0), -3), (dict(hd=96), -3), (dict(page=24), -3), (dict(page=0), -3), (dict(page=1 << 17), -3),
              (dict(block=3), -3), (dict(block=32), -3), (dict(block=0), -3), (dict(n_pages=0), -3), (dict(KV=0), -3),
              (dict(k=None), -3), (dict(v_scale=None), -3), (dict(k=(1 << 20) + 8), -3), (dict(k_scale=(1 << 20) + 2), -3),
              (dict(n_pages=1 << 28), -5)]
BAD_BATCHES = [dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(n_seq=0), dict(n_seq=70000),
               dict(table_stride=0), dict(total_q=-1), dict(max_q=-1), dict(max_kv=-1)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_refuses_bad_caches(kw, code):
    L = _lib.load()
    c, b, s = c_cache(**kw), c_batch(), c_score()
    assert L.tlmg_kv8_append(C.byref(c), C.byref(b), 0, 1 << 20, 1 << 20, 0, 1) == code
    assert L.tlmg_kv8_read(C.byref(c), 1, 1 << 20, 4, 1 << 20, 1 << 20, 4, 1 << 20, 1 << 20, 1) == code
    assert L.tlmg_kv8_attend(C.byref(c), C.byref(b), C.byref(s), 4, 0, 1 << 20, 0, 1 << 20, None, None, 0, 1 << 20, 1 << 30, 1) == code
    assert L.tlmg_kv8_attend_work_bytes(C.byref(c), C.byref(b), C.byref(s), 4, 0, 0) == 0
    assert L.tlmg_kv8_compact(C.byref(c), C.byref(c_cache()), 1, 1 << 20, 4, 1 << 20, 1 << 20, 4, 1 << 20, 8, None, 0, None, 0, 1) == code
    assert len(L.tlmg_errmsg()) > 10


@pytest.mark.parametrize("kw", BAD_BATCHES)
def test_refuses_bad_batches(kw):
    L = _lib.load()
    c, b, s = c_cache(), c_batch(**kw), c_score()
    assert L.tlmg_kv8_append(C.byref(c), C.byref(b), 0, 1 << 20, 1 << 20, 0, 1) == -3
    assert L.tlmg_kv8_attend(C.byref(c), C.byref(b), C.byref(s), 4, 0, 1 << 20, 0, 1 << 20, None, None, 0, 1 << 20, 1 << 30, 1) == -3


def test_refuses_bad_calls():
    L = _lib.load()
    c, b, s = c_cache(), c_batch(), c_score()
    ok = 1 << 20

    def attend(c=c, b=b, s=s, H=4, dt=0, q=ok, st=0, out=ok, w=None, ws=0, work=ok, wb=1 << 30):
        return L.tlmg_kv8_attend(C.byref(c), C.byref(b), C.byref(s), H, dt, q, st, out, None, w, ws, work, wb, 1)

    assert attend(H=3) == -3 and attend(H=34) == -3 and attend(H=0) == -3
    assert attend(dt=8) == -3 and attend(q=None) == -3 and attend(out=None) == -3
    assert attend(q=ok + 4) == -3 and attend(out=ok + 8) == -3
    assert attend(st=100) == -3 and attend(st=4 * 64 + 2) == -3 and attend(dt=1, st=4 * 64 + 4) == -3
    assert attend(w=ok, ws=39) == -3 and attend(w=ok, ws=40, b=c_batch(max_q=65)) == -3
    assert attend(w=ok, ws=40, wb=64) == -5 and attend(w=ok, ws=40, work=None) == -3 and attend(w=ok, ws=40, work=ok + 4) == -3
    for kw in (dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0),
               dict(softcap=float("inf")), dict(window=-1), dict(doc=ok, doc_stride=0)):
        assert attend(s=c_score(**kw)) == -3, kw
    assert attend(b=c_batch(total_q=1 << 30)) == -5
    assert attend(b=c_batch(total_q=0)) == 0 and attend(b=c_batch(max_q=0)) == 0
    app = lambda dt=0, k=ok, st=0: L.tlmg_kv8_append(C.byref(c), C.byref(b), dt, k, ok, st, 1)  # noqa: E731
    assert app(dt=12) == -3 and app(k=None) == -3 and app(k=ok + 4) == -3 and app(st=64) == -3 and app(st=2 * 64 + 1) == -3
    sel = lambda n=1, mk=40, ws=40, keep=8, a=2, r=2, w=ok: L.tlmg_kv8_select(n, 2, ok, mk, w, ws, keep, a, r, ok, ok, 1)  # noqa: E731
    assert sel(n=0) == -3 and sel(ws=39) == -3 and sel(keep=0) == -3 and sel(a=7) == -3 and sel(a=-1) == -3 and sel(r=-1) == -3
    assert sel(w=None) == -3
    cmp_ = lambda d, keep=8, wo=None, ws=8: L.tlmg_kv8_compact(C.byref(c), C.byref(d), 1, ok, 4, ok, ok, 4, ok, keep, None, 0, wo, ws, 1)  # noqa: E731
    assert cmp_(c_cache(hd=128)) == -3 and cmp_(c_cache(KV=4)) == -3 and cmp_(c_cache(pos=None)) == -3
    assert cmp_(c_cache(), keep=0) == -3 and cmp_(c_cache(), wo=ok) == -3
    rd = lambda n=1, st=4, tot=4, k=ok: L.tlmg_kv8_read(C.byref(c), n, ok, st, ok, ok, tot, k, ok, 1)  # noqa: E731
    assert rd(n=0) == -3 and rd(st=0) == -3 and rd(tot=-1) == -3 and rd(k=None) == -3 and rd(k=ok + 4) == -3 and rd(tot=0) == 0


def test_wrapper_refuses_host_tensors_and_shapes():
    k = torch.zeros((2, 2, 16, 64), dtype=torch.int8)
    s = torch.zeros((2, 2, 1))
    with pytest.raises(TlmError) as e:
        K.Kv8Cache.from_pools(k, k, s, s)
    assert e.value.code == -3
    with pytest.raises(TlmError):
        K.Kv8Cache.from_pools(k.float(), k.float(), s, s)
    with pytest.raises(TlmError):
        K.Kv8Cache(2, 2, 16, 64, block=3, device="cpu")
    with pytest.raises(TlmError):
        K.Kv8Cache(2, 2, 16, 64, fmt=5, device="cpu")


# ---- append and read (GPU) -----------------------------------------------------------
def same(a, b):
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    return ((a.view(np.uint32) == b.view(np.uint32)) | (np.isnan(a) & np.isnan(b))).all()


def assert_cache(cache, host):
    assert (cache.k.view(torch.uint8).cpu().numpy() == host.k).all()
    assert (cache.v.view(torch.uint8).cpu().numpy() == host.v).all()
    assert same(cache.k_scale.cpu().numpy(), host.ks) and same(cache.v_scale.cpu().numpy(), host.vs)
    if host.pos is not None:
        assert (cache.pos.cpu().numpy() == host.pos).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [K.INT8, K.E4M3])
@pytest.mark.parametrize("KV,hd,page,block", [(2, 64, 16, 16), (4, 128, 64, 16), (1, 256, 32, 8), (3, 128, 1, 1),
                                              (2, 128, 256, 256), (5, 64, 8, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_append_bits(fmt, KV, hd, page, block, dtype):
    """Prompts and single tokens in turn, from any row on: the pools equal the
    restatement's byte for byte, rows of begun blocks rounded again included."""
    rng = np.random.default_rng(7)
    lens = np.array([0, 0, 0, 0])
    cap = [3 * block + 70, 40, 200, 1]
    table, n_pages = tables(rng, cap, page)
    host = Host(n_pages, KV, page, hd, fmt, block, True, 3)
    cache = host.gpu()
    for step, news in enumerate([(block + 5, 1, 0, 1), (1, 1, 17, 0), (1, 0, 1, 0), (0, 2, 100, 0), (50, 30, 1, 0), (1, 1, 1, 0)]):
        lens = lens + np.array(news)
        q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        n = int(q_start[-1])
        x = [torch.from_numpy((rng.standard_normal((n, KV, hd)) * 10 ** rng.uniform(-2, 2, (n, KV, 1))).astype(np.float32)).to(dtype) for _ in range(2)]
        q_pos = rng.integers(0, 1 << 30, n).astype(np.int32) if step % 2 else None
        cache.append(x[0].cuda(), x[1].cuda(), batch(table, q_start, lens, q_pos))
        host.append(x[0].float().numpy(), x[1].float().numpy(), table, q_start, lens, q_pos)
        assert_cache(cache, host)
    row0 = np.array([3, 0, 5, 0], np.int32)
    n = lens - row0
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    k, v = cache.read(up(table), up(row0), up(start), int(start[-1]))
    for s in range(4):
        for got, which in ((k, "k"), (v, "v")):
            want = host.rows(which, table[s], lens[s])[row0[s]:].astype(np.float32)
            assert same(got[start[s]:start[s + 1]].cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [K.INT8, K.E4M3])
def test_append_special_values(fmt):
    """Zeros, subnormals, the largest floats, ties, infinities and NaN."""
    rng = np.random.default_rng(1)
    KV, hd, page, block = 1, 64, 16, 4
    x = np.zeros((32, KV, hd), np.float32)
    x[4:8] = rng.standard_normal((4, KV, hd)) * 1e-42
    x[8:12] = np.float32(3.4e38) * rng.uniform(-1, 1, (4, KV, hd)).astype(np.float32)
    x[12:16] = (np.arange(256).reshape(4, 1, 64) - 127.5)
    x[13, 0, 0] = 127
    x[16:20] = rng.standard_normal((4, KV, hd))
    x[17, 0, 3] = np.nan
    x[20:24, 0, 5] = np.inf
    x[24:28] = 448 * rng.uniform(-1, 1, (4, KV, hd))
    x[28] = -x[27]
    table = np.array([[1, 0]], np.int32)
    host = Host(3, KV, page, hd, fmt, block, False, 0)
    cache = host.gpu()
    for lo, hi in ((0, 30), (30, 32)):
        qs = np.array([0, hi - lo], np.int32)
        cache.append(up(x[lo:hi]), up(-x[lo:hi]), batch(table, qs, [hi]))
        host.append(x[lo:hi], -x[lo:hi], table, qs, [hi])
        assert_cache(cache, host)
    assert np.isnan(host.ks).sum() >= 2


@pytest.mark.gpu
def test_append_strides_and_bad_sequences():
    """Rows inside a wider tensor; sequences whose lengths do not fit and pages out of range write nothing."""
    rng = np.random.default_rng(2)
    KV, hd, page = 2, 64, 16
    fused = torch.from_numpy(rng.standard_normal((9, 8, hd)).astype(np.float32)).cuda()   # q | k | v heads of a token
    table = np.array([[3, 4], [0, 99], [1, -1], [2, 5]], np.int32)
    host = Host(6, KV, page, hd, K.INT8, 16, False, 1)
    cache = host.gpu()
    qs = np.array([0, 2, 4, 6, 9], np.int32)
    lens = np.array([20, 18, 40, 2], np.int32)   # 2: more rows than the table holds; 3: fewer rows than new tokens
    cache.append(fused[:, 4:6], fused[:, 6:8], batch(table, qs, lens))
    k, v = fused[:, 4:6].cpu().numpy(), fused[:, 6:8].cpu().numpy()
    host.append(k, v, table[:1], qs[:2], lens[:1])
    # sequence 1: rows 16 and 17 lie on page 99
    assert_cache(cache, host)
    odd = torch.empty(9 * 2 * hd + 1, device="cuda")[1:].view(9, 2, hd)     # off 16 bytes: copied
    odd.copy_(fused[:, 4:6])
    cache2 = Host(6, KV, page, hd, K.INT8, 16, False, 1).gpu()
    cache2.append(odd, fused[:, 6:8], batch(table[:1], qs[:2], lens[:1]))
    assert (cache2.k == cache.k).all() and (cache2.v == cache.v).all()
    k, v = cache.read(up(table), up(np.array([18, 0, 0, 0])).int(), up(np.array([0, 2, 4, 4, 4])).int(), 4)
    assert torch.isnan(k[:2]).all()      # they continue a block whose scale was NaN: it stays
    far, _ = cache.read(up(table[1:2]), up(np.array([16])).int(), up(np.array([0, 30])).int(), 30)
    assert torch.isnan(far).all()


# ---- attention (GPU) -------------------------------------------------------------------
DECODE = [   # (lens, news, H, KV, hd, page, block)
    ([1], [1], 8, 2, 64, 16, 16), ([2, 1, 33], [1, 1, 1], 4, 4, 64, 16, 1), ([300, 31, 32, 64], [1, 1, 1, 1], 32, 4, 128, 64, 16),
    ([701], [1], 32, 4, 128, 16, 8), ([97, 500], [1, 1], 6, 2, 128, 32, 32), ([130], [1], 5, 1, 256, 1, 1),
    ([260, 5], [1, 1], 32, 2, 64, 8, 8), ([1500], [1], 16, 1, 128, 256, 64), ([40, 0, 7], [1, 0, 1], 10, 2, 64, 16, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", [K.INT8, K.E4M3])
@pytest.mark.parametrize("case", DECODE)
def test_decode(case, fmt, dtype):
    lens, news, H, KV, hd, page, block = case
    host, table, q_start, q, _ = make(11, lens, news, H, KV, hd, fmt, page, block, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,news,H,KV,hd", [([90, 33, 5], [5, 33, 1], 8, 2, 64), ([70], [70], 6, 2, 128), ([200, 7], [3, 0], 7, 1, 64),
                                               ([150], [40], 4, 2, 256)])
def test_few_and_many_tokens(lens, news, H, KV, hd, dtype):
    host, table, q_start, q, _ = make(12, lens, news, H, KV, hd, K.INT8, 32, 8, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H)
    check_attend(host, table, q_start, lens, q, H, causal=False)


MANY = [   # (lens, news, H, KV, hd, page, block): more query rows per KV head than a tensor-core tile
    ([300, 40, 7], [300, 40, 7], 8, 2, 64, 16, 16), ([500], [130], 4, 4, 128, 64, 16), ([129, 260], [128, 129], 3, 1, 64, 8, 1),
    ([257], [257], 6, 2, 128, 32, 32), ([400, 1], [16, 0], 32, 2, 128, 256, 64), ([640], [40], 16, 1, 64, 1, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", [K.INT8, K.E4M3])
@pytest.mark.parametrize("case", MANY)
def test_prefill(case, fmt, dtype):
    lens, news, H, KV, hd, page, block = case
    host, table, q_start, q, _ = make(31, lens, news, H, KV, hd, fmt, page, block, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H)
    check_attend(host, table, q_start, lens, q, H, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("name", ["cap", "cap_small", "alibi", "alibi_both", "window", "window_one", "sinks", "prefix", "prefix_all", "doc",
                                  "doc_jumbled", "doc_short", "all", "scale", "window_open"])
def test_prefill_score_shapes(name, dtype):
    lens, news, H, KV, hd = [290, 180, 20], [200, 180, 3], 4, 2, 64
    host, table, q_start, q, rng = make(32, lens, news, H, KV, hd, K.E4M3, 16, 4, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H, **mods_of(name, rng, lens, H))


@pytest.mark.gpu
def test_prefill_positions_and_poison():
    """The position pool, masked rows with NaN scales, rows without keys and bad sequences at prefill sizes."""
    lens, news, H, KV, hd = [300, 200], [150, 140], 4, 2, 128
    host, table, q_start, q, rng = make(33, lens, news, H, KV, hd, K.INT8, 16, 16, pos=True, dtype=torch.bfloat16)
    for s, L in enumerate(lens):
        for t in range(L):
            host.pos[table[s, t // 16], :, t % 16] = rng.integers(0, 500, KV)
    q_pos = rng.integers(0, 500, 290).astype(np.int32)
    q_pos[:3] = [0, 499, 0]
    host.pos[table[0, 3]] = 1000                       # never seen (causal)
    host.ks[table[0, 3]], host.vs[table[0, 3]] = np.nan, np.nan
    host.vs[table[1, 2]] = 1e25                        # seen by few
    host.pos[table[1, 2]] = 498
    check_attend(host, table, q_start, lens, q, H, q_pos=q_pos)
    check_attend(host, table, q_start, lens, q, H, q_pos=q_pos, window=40)
    good = host.gpu().attend(q.cuda(), batch(table, q_start, lens, q_pos))
    out, lse = host.gpu().attend(q.cuda(), batch(table, q_start, [300, 4000], q_pos, max_kv=300), lse=True)
    assert torch.isnan(out[150:]).all() and torch.isnan(lse[150:]).all() and (out[:150] == good[:150]).all()
    bad = table.copy()
    bad[1, 4] = -5                                     # positions there are unknown: every query that may see position 0
    out = host.gpu().attend(q.cuda(), batch(bad, q_start, lens, q_pos))
    assert torch.isnan(out[150:]).all() and (out[:150] == good[:150]).all()


# A bound on the rows by which these calls count as large: the kernels for many query rows take them, small as they are.
WIDE = 60000


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", [K.INT8, K.E4M3])
@pytest.mark.parametrize("case", MANY)
def test_wide(case, fmt, dtype):
    lens, news, H, KV, hd, page, block = case
    host, table, q_start, q, _ = make(31, lens, news, H, KV, hd, fmt, page, block, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H, max_kv=WIDE)
    check_attend(host, table, q_start, lens, q, H, max_kv=WIDE, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("news", [[200, 180, 3], [90, 40, 20]])
@pytest.mark.parametrize("name", ["cap", "cap_small", "alibi", "alibi_both", "window", "window_one", "sinks", "prefix", "prefix_all", "doc",
                                  "doc_jumbled", "doc_short", "all", "scale", "window_open"])
def test_wide_score_shapes(name, news, dtype):
    lens, H, KV, hd = [290, 180, 20], 4, 2, 64
    host, table, q_start, q, rng = make(32, lens, news, H, KV, hd, K.E4M3, 16, 4, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H, max_kv=WIDE, **mods_of(name, rng, lens, H))


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[150, 140], [290, 195]])
def test_wide_positions_and_poison(news):
    """The position pool, masked rows with NaN scales, rows without keys and bad sequences."""
    lens, H, KV, hd = [300, 200], 4, 2, 128
    n, n0 = sum(news), news[0]
    host, table, q_start, q, rng = make(33, lens, news, H, KV, hd, K.INT8, 16, 16, pos=True, dtype=torch.bfloat16)
    for s, L in enumerate(lens):
        for t in range(L):
            host.pos[table[s, t // 16], :, t % 16] = rng.integers(0, 500, KV)
    q_pos = rng.integers(0, 500, n).astype(np.int32)
    q_pos[:3] = [0, 499, 0]
    host.pos[table[0, 3]] = 1000                       # never seen (causal)
    host.ks[table[0, 3]], host.vs[table[0, 3]] = np.nan, np.nan
    host.vs[table[1, 2]] = 1e25                        # seen by few
    host.pos[table[1, 2]] = 498
    check_attend(host, table, q_start, lens, q, H, q_pos=q_pos, max_kv=WIDE)
    check_attend(host, table, q_start, lens, q, H, q_pos=q_pos, max_kv=WIDE, window=40)
    good = host.gpu().attend(q.cuda(), batch(table, q_start, lens, q_pos, max_kv=WIDE))
    out, lse = host.gpu().attend(q.cuda(), batch(table, q_start, [300, 70000], q_pos, max_kv=WIDE), lse=True)
    assert torch.isnan(out[n0:]).all() and torch.isnan(lse[n0:]).all() and (out[:n0] == good[:n0]).all()
    bad = table.copy()
    bad[1, 4] = -5                                     # positions there are unknown: every query that may see position 0
    out = host.gpu().attend(q.cuda(), batch(bad, q_start, lens, q_pos, max_kv=WIDE))
    assert torch.isnan(out[n0:]).all() and (out[:n0] == good[:n0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("pool", ["ascending", "jumbled_tiles", "none"])
@pytest.mark.parametrize("name", ["causal", "window", "sinks", "doc", "doc_window", "both_ways"])
def test_prefill_whole_tiles(name, pool, dtype):
    """Key tiles that every query sees, that none sees and that some see, by positions with gaps and by documents."""
    lens, news, H, KV, hd = [700, 420], [260, 150], 4, 2, 64
    host, table, q_start, q, rng = make(34, lens, news, H, KV, hd, K.INT8, 16, 16, pos=pool != "none", dtype=dtype)
    q_pos = None
    if pool != "none":
        q_pos = np.zeros(q_start[-1], np.int32)
        for s, L in enumerate(lens):
            for h in range(KV):                        # every head has kept other rows
                p = np.sort(rng.permutation(2 * L)[:L]).astype(np.int32)
                p[L - news[s]:] = 2 * L + np.arange(news[s])
                if pool == "jumbled_tiles":            # whole tiles of 128 rows, the queries' own among them, in another order
                    p = p[np.concatenate([np.arange(128, 256), np.arange(L - L % 128, L), np.arange(128),
                                          np.arange(256, L - L % 128)])]
                for t in range(L):
                    host.pos[table[s, t // 16], h, t % 16] = p[t]
            q_pos[q_start[s]:q_start[s + 1]] = 2 * L + np.arange(news[s])
    span = 2 * max(lens) + 300
    doc = np.zeros((2, span), np.int32)
    doc[:, span // 3:], doc[:, span // 2:] = 1, 2
    doc[0, :] = np.where(np.arange(span) < 600, doc[0, :], 2)
    mods = {"causal": {}, "window": dict(window=300), "sinks": dict(window=140, prefix=np.array([130, 3], np.int32)), "doc": dict(doc=doc),
            "doc_window": dict(doc=doc, window=200), "both_ways": dict(causal=False)}[name]
    check_attend(host, table, q_start, lens, q, H, q_pos=q_pos, max_kv=WIDE, **mods)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("max_q,max_kv", [(600, 310), (40000, 200000), (40000, 60000)])
def test_prefill_loose_bounds(max_q, max_kv, dtype):
    """max_q and max_kv far above the lengths, by which the work is divided: all, some or one of the KV heads in a turn."""
    lens, news, H, KV, hd = [300, 5, 260], [280, 5, 3], 6, 3, 128
    host, table, q_start, q, _ = make(35, lens, news, H, KV, hd, K.E4M3, 16, 16, dtype=dtype)
    out, lse = host.gpu().attend(q.cuda(), batch(table, q_start, lens, max_q=max_q, max_kv=max_kv), lse=True)
    ref, rlse, _, ds, mags, _ = reference(host, q.float().numpy(), table, q_start, lens, H)
    assert_close(out.float().cpu().numpy(), ref, out_bound(ref, mags, ds, dtype))
    assert_close(lse.cpu().numpy(), rlse, ds + 2.0 ** -18 + 2.0 ** -22 * np.abs(rlse))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("news", [[40, 33], [200, 7]])
@pytest.mark.parametrize("name", ["plain", "window", "sinks", "doc", "cap", "both_ways"])
def test_prefill_pieces(name, news, dtype):
    """Few query tiles over many rows: the keys go in pieces that are joined, some of them without a visible key."""
    lens, H, KV, hd, bound = [2600, 1100], 12, 2, 64, 30000
    host, table, q_start, q, rng = make(36, lens, news, H, KV, hd, K.INT8, 64, 16, dtype=dtype)
    doc = np.zeros((2, max(lens)), np.int32)
    doc[:, 900:], doc[0, 2480:] = 1, 2
    mods = {"plain": {}, "window": dict(window=700), "sinks": dict(window=150, prefix=np.array([600, 20], np.int32)), "doc": dict(doc=doc),
            "cap": dict(softcap=3.0), "both_ways": dict(causal=False)}[name]
    check_attend(host, table, q_start, lens, q, H, max_kv=bound, **mods)


@pytest.mark.gpu
def test_long_prompt():
    """A prompt of more query tiles than a grid's second dimension takes: its last tokens as a call of their own gives them.
    Both are within (2^-8 + 2^-10) max |v| of the exact result."""
    L, H, KV, hd, last = 16500, 32, 2, 64, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randn((L, h, hd), generator=g, device="cuda").to(torch.bfloat16) for h in (KV, KV, H))
    cache = K.Kv8Cache(-(-L // 64), KV, 64, hd)
    table = np.arange(-(-L // 64), dtype=np.int32)[None]
    whole = batch(table, [0, L], [L])
    cache.append(k, v, whole)
    out = cache.attend(q, whole)[L - last:].float()
    want = cache.attend(q[L - last:].contiguous(), batch(table, [0, last], [L])).float()
    assert float((out - want).abs().max()) <= 2 * (2.0 ** -8 + 2.0 ** -10) * float(v.float().abs().max())


def mods_of(name, rng, lens, H):
    n = len(lens)
    doc = np.full((n, max(lens)), -1, np.int32)
    for s, L in enumerate(lens):
        doc[s, :L] = np.sort(rng.integers(0, 3, L))
    jumbled = rng.permutation(doc.reshape(-1)).reshape(doc.shape).astype(np.int32)
    slopes = (2.0 ** -np.linspace(0.5, 8, H)).astype(np.float32)
    return {"cap": dict(softcap=5.0), "cap_small": dict(softcap=0.25), "alibi": dict(slopes=slopes),
            "alibi_both": dict(slopes=slopes, causal=False), "window": dict(window=20), "window_one": dict(window=1),
            "sinks": dict(window=9, prefix=np.arange(1, n + 1, dtype=np.int32) * 3), "prefix": dict(prefix=np.array([L // 2 for L in lens], np.int32)),
            "prefix_all": dict(prefix=np.array([L + 9 for L in lens], np.int32)), "doc": dict(doc=doc), "doc_jumbled": dict(doc=jumbled, causal=False),
            "doc_short": dict(doc=np.ascontiguousarray(doc[:, :5])), "all": dict(softcap=8.0, slopes=slopes, window=50, prefix=np.full(n, 4, np.int32), doc=doc),
            "scale": dict(scale=0.4), "window_open": dict(window=12, causal=False)}[name]


MODS = ["cap", "cap_small", "alibi", "alibi_both", "window", "window_one", "sinks", "prefix", "prefix_all", "doc", "doc_jumbled",
        "doc_short", "all", "scale", "window_open"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", MODS)
def test_score_shapes(name, dtype):
    lens, news, H, KV, hd = [150, 64, 9], [7, 1, 9], 6, 2, 64
    host, table, q_start, q, rng = make(13, lens, news, H, KV, hd, K.E4M3, 16, 4, dtype=dtype)
    check_attend(host, table, q_start, lens, q, H, weights=True, **mods_of(name, rng, lens, H))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["window", "alibi", "sinks", "doc", "prefix"])
def test_positions_pool(name):
    """Rows at positions of their own per head, in no order; explicit query positions."""
    lens, news, H, KV, hd = [100, 40], [3, 1], 8, 2, 128
    host, table, q_start, q, rng = make(14, lens, news, H, KV, hd, K.INT8, 16, 16, pos=True)
    for s, L in enumerate(lens):
        for t in range(L):
            host.pos[table[s, t // 16], :, t % 16] = rng.integers(0, 160, KV)
    mods = mods_of(name, rng, [160, 160], H)
    check_attend(host, table, q_start, lens, q, H, q_pos=np.array([60, 159, 3, 80], np.int32), weights=True, **mods)


@pytest.mark.gpu
def test_query_positions_without_pool():
    """Query positions other than the last rows' (an earlier position asked again, one past the end)."""
    lens, news, H, KV, hd = [120, 70], [4, 2], 4, 2, 64
    host, table, q_start, q, rng = make(15, lens, news, H, KV, hd)
    q_pos = np.array([0, 119, 50, 2147483647, 200, 33], np.int32)
    check_attend(host, table, q_start, lens, q, H, q_pos=q_pos, weights=True)
    check_attend(host, table, q_start, lens, q, H, q_pos=np.array([0, 119, 50, 90, 75, 33], np.int32), window=30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_keys(dtype):
    """Queries that see nothing: 0 and -inf, whatever the masked rows hold (NaN scales, any codes)."""
    lens, news, H, KV, hd = [64, 40], [3, 2], 4, 2, 64
    host, table, q_start, q, _ = make(16, lens, news, H, KV, hd, K.E4M3, 16, 16, dtype=dtype)
    doc = np.zeros((2, 64), np.int32)
    doc[0, 61:] = [5, 0, 6]          # the second query's document is the first rows'
    doc[1, :20] = 1                  # rows 0..15 of sequence 1 are masked: make them poison
    host.ks[table[1, 0]] = np.nan
    host.vs[table[1, 0]] = np.inf
    host.k[table[1, 0]] = 0x7F
    host.v[table[1, 0]] = 0xFF
    doc[0, 61], doc[0, 63] = -3, 77
    doc[0, 61] = 9
    q_pos = np.array([200, 62, 300, 38, 39], np.int32)   # past the document table: document -1, which no key has
    score = dict(doc=doc, q_pos=q_pos)
    out, lse = check_attend(host, table, q_start, lens, q, H, weights=True, **score)
    assert (out[0] == 0).all() and (out[2] == 0).all() and torch.isinf(lse[0]).all() and torch.isfinite(out).all()
    # the same rows seen: NaN, and only for the queries that see them
    out = host.gpu().attend(q.cuda(), batch(table, q_start, lens))
    assert torch.isfinite(out[:3].float()).all() and torch.isnan(out[3:].float()).all()


@pytest.mark.gpu
def test_scales_far_apart():
    """A masked or unimportant row's scale of 1e30 or 1e-30 costs the others no precision; large and tiny queries."""
    lens, news, H, KV, hd = [200], [2], 4, 1, 64
    host, table, q_start, q, rng = make(17, lens, news, H, KV, hd, K.INT8, 16, 4, spread=3.0)
    doc = np.ones((1, 200), np.int32)
    doc[0, 40:44] = 0
    host.vs[table[0, 2], :, 2] = 1e30
    host.ks[table[0, 2], :, 2] = 1e30
    host.vs[table[0, 5], :, 1] = 1e-30
    host.ks[table[0, 6], :, 1] = 1e-30
    for mul in (1.0, 1e-20, 30.0):
        check_attend(host, table, q_start, lens, q * mul, H, doc=doc)
    host.vs[table[0, 2], :, 2] = 1e4
    host.ks[table[0, 2], :, 2] = 1e-3
    check_attend(host, table, q_start, lens, q, H)


@pytest.mark.gpu
def test_bad_pages_and_lengths():
    """Out-of-range page entries and lengths that break the bounds: NaN for who is concerned, others untouched."""
    lens, news, H, KV, hd = [50, 50, 50], [2, 2, 2], 4, 2, 64
    host, table, q_start, q, _ = make(18, lens, news, H, KV, hd)
    good = host.gpu().attend(q.cuda(), batch(table, q_start, lens))
    bad = table.copy()
    bad[1, 2] = 1 << 20
    out, lse = host.gpu().attend(q.cuda(), batch(bad, q_start, lens), lse=True)
    assert (out[:2] == good[:2]).all() and (out[4:] == good[4:]).all() and torch.isnan(out[2:4]).all() and torch.isnan(lse[2:4]).all()
    out = host.gpu().attend(q.cuda(), batch(bad, q_start, lens), K.Score(window=1))     # rows 32..47 are not seen
    assert torch.isfinite(out).all()
    for L in (1, 65, 1000):      # fewer rows than tokens; more than max_kv; more than the table
        out, lse = host.gpu().attend(q.cuda(), batch(table, q_start, [50, L, 50], max_kv=64), lse=True)
        assert (out[:2] == good[:2]).all() and (out[4:] == good[4:]).all() and torch.isnan(out[2:4]).all() and torch.isnan(lse[2:4]).all()
    w = torch.zeros((3, KV, 64), device="cuda")
    host.gpu().attend(q.cuda(), batch(table, q_start, [50, 65, 50], max_kv=64), weights=w)
    assert (w[1] == 0).all() and (w[0].sum() - 2 * H < 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_long_context_and_repeat(dtype):
    """A context over many spans; the same bits in every run, on another stream and with a larger max_kv within rounding."""
    lens, news, H, KV, hd = [5000, 3], [1, 1], 8, 2, 64
    host, table, q_start, q, _ = make(19, lens, news, H, KV, hd, K.INT8, 64, 16, dtype=dtype)
    a, _ = check_attend(host, table, q_start, lens, q, H, weights=True)
    cache, b, qd = host.gpu(), batch(table, q_start, lens), q.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = [cache.attend(qd, b) for _ in range(3)]
    s.synchronize()
    assert all((x == a).all() for x in c)


@pytest.mark.gpu
def test_query_strides():
    """q as the leading heads of a fused q|k|v tensor, and off alignment (copied)."""
    lens, news, H, KV, hd = [80], [5], 8, 2, 64
    host, table, q_start, q, _ = make(20, lens, news, H, KV, hd)
    cache, b = host.gpu(), batch(table, q_start, lens)
    want = cache.attend(q.cuda(), b)
    fused = torch.zeros((5, H + 2 * KV, hd), device="cuda")
    fused[:, :H] = q.cuda()
    assert (cache.attend(fused[:, :H], b) == want).all()
    heads_apart = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert (cache.attend(heads_apart, b) == want).all()
    odd = torch.empty(5 * H * hd + 1, device="cuda")[1:].view(5, H, hd)
    odd.copy_(q)
    assert (cache.attend(odd, b) == want).all()


@pytest.mark.gpu
def test_pools_past_32_bits():
    """Rows whose byte offsets pass 2^32: append, read, attend and evict at the pool's end."""
    KV, hd, page, n_pages = 4, 256, 1024, 4400          # 4.6 GB of K codes
    cache = K.Kv8Cache(n_pages, KV, page, hd, K.INT8, 64, positions=True)
    rng = np.random.default_rng(3)
    L, H = 100, 8
    table = np.array([[n_pages - 1]], np.int32)
    x = rng.standard_normal((2, L, KV, hd)).astype(np.float32)
    qs = np.array([0, L], np.int32)
    cache.append(up(x[0]), up(x[1]), batch(table, qs, [L]))
    k, v = cache.read(up(table), up(np.array([0])).int(), up(qs), L)
    assert float((k.cpu() - torch.from_numpy(x[0])).abs().max()) < 0.03
    host = Host(1, KV, page, hd, K.INT8, 64, True, 3)
    host.append(x[0], x[1], np.array([[0]]), qs, [L])
    q = rng.standard_normal((1, H, hd)).astype(np.float32)
    out = cache.attend(up(q), batch(table, np.array([0, 1]), [L]))
    want, _, _, ds, mag, _ = reference(host, q, np.array([[0]]), [0, 1], [L], H)
    assert_close(out.cpu().numpy(), want, out_bound(want, mag, ds, torch.float32))
    w = torch.rand((1, KV, L), device="cuda")
    rows, lens = cache.evict(w, batch(table, np.array([0, 1]), [L]), up(np.array([[n_pages - 2]], np.int32)), 40, 4, 8)
    assert int(lens) == 40 and (cache.pos[n_pages - 2, :, :40] == rows[0]).all()


# ---- eviction (GPU) -----------------------------------------------------------------------
def select_reference(w, L, keep, sink, recent):
    if L <= keep:
        return np.arange(L)
    w = np.where(np.isnan(w[:L]), -np.inf, w[:L].astype(np.float64))
    nan = np.isnan(w)
    t = np.arange(L)
    held = (t < sink) | (t >= L - recent)
    return np.sort(np.lexsort((t, -w, nan, ~held))[:keep])


@pytest.mark.gpu
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (50, 4, 10), (64, 64, 0), (100, 0, 100), (700, 1, 2), (2000, 0, 0)])
def test_select(keep, sink, recent):
    rng = np.random.default_rng(5)
    lens = np.array([0, 1, 49, 50, 51, 700, 1500, 5000], np.int32)
    KV = 2
    w = rng.random((len(lens), KV, 5003)).astype(np.float32)
    w[5] = np.round(w[5], 1)                    # many ties
    w[6, 0] = 0.25                              # nothing but ties
    w[6, 1, ::3] = np.nan
    w[7] = (w[7] - 0.5) * 10.0 ** rng.integers(-40, 38, w[7].shape)
    w[7, :, ::7] = 0.0
    w[7, :, 3::7] = -0.0
    w[7, 0, 10] = np.inf
    w[7, 0, 11] = -np.inf
    rows = torch.empty((len(lens), KV, keep), dtype=torch.int32, device="cuda")
    out = torch.empty(len(lens), dtype=torch.int32, device="cuda")
    wd, ld = up(w), up(lens)
    _lib.check(_lib.load().tlmg_kv8_select(len(lens), KV, ld.data_ptr(), 5003, wd.data_ptr(), 5003, keep, sink, recent, rows.data_ptr(),
                                           out.data_ptr(), 1))
    rows = rows.cpu().numpy()
    assert (out.cpu().numpy() == np.minimum(lens, keep)).all()
    for s, L in enumerate(lens):
        for h in range(KV):
            want = select_reference(w[s, h], int(L), keep, sink, recent)
            assert (rows[s, h, :len(want)] == want).all() and (rows[s, h, len(want):] == -1).all(), (s, h)


@pytest.mark.gpu
@pytest.mark.parametrize("src_fmt,dst_fmt", [(K.INT8, K.INT8), (K.E4M3, K.E4M3), (K.INT8, K.E4M3), (K.E4M3, K.INT8)])
@pytest.mark.parametrize("hd,page,block,dpage,dblock,pos", [(64, 16, 16, 16, 16, True), (128, 32, 8, 64, 32, False), (256, 8, 1, 16, 4, True)])
def test_evict_bits(src_fmt, dst_fmt, hd, page, block, dpage, dblock, pos):
    """Kept rows stored again in another cache: codes, scales, positions and weights equal the restatement's."""
    rng = np.random.default_rng(6)
    lens, KV, keep, sink, recent = [200, 33, 7, 0], 2, 50, 3, 9
    host, table, _, _, _ = make(21, lens, [0, 0, 0, 0], 2, KV, hd, src_fmt, page, block, pos)
    w = rng.random((4, KV, 210)).astype(np.float32)
    dtable, n_dst = tables(rng, [min(L, keep) for L in lens], dpage)
    dst = Host(n_dst, KV, dpage, hd, dst_fmt, dblock, True, 9)
    src_gpu, dst_gpu = host.gpu(), dst.gpu()
    w_out = torch.full((4, KV, keep + 2), 7.0, device="cuda")
    rows, new = src_gpu.evict(up(w), batch(table, [0, 0, 0, 0, 0], lens, max_q=1), up(dtable), keep, sink, recent, dst=dst_gpu, weights_out=w_out)
    want_w = np.full((4, KV, keep + 2), 7.0, np.float32)
    for s, L in enumerate(lens):
        assert int(new[s]) == min(L, keep)
        kr, vr, pr = host.rows("k", table[s], L), host.rows("v", table[s], L), host.positions(table[s], L)
        for h in range(KV):
            r = select_reference(w[s, h], L, keep, sink, recent)
            assert (rows[s, h].cpu().numpy()[:len(r)] == r).all()
            want_w[s, h, :keep] = 0
            want_w[s, h, :len(r)] = w[s, h, r]
            for j0 in range(0, len(r), dblock):
                rr = r[j0:j0 + dblock]
                e, o = dtable[s, j0 // dpage], j0 % dpage
                for x, codes, scale in ((kr, dst.k, dst.ks), (vr, dst.v, dst.vs)):
                    c, d = quantise(x[rr, h].astype(np.float32), dst_fmt)
                    codes[e, h, o:o + len(rr)], scale[e, h, o // dblock] = c, d
                dst.pos[e, h, o:o + len(rr)] = pr[rr, h]
    assert_cache(dst_gpu, dst)
    assert_cache(src_gpu, host)
    assert (w_out.cpu().numpy() == want_w).all()


@pytest.mark.gpu
def test_evict_then_decode():
    """The whole path: decode with accumulated weights, eviction in the same pools, append and decode on the evicted rows."""
    rng = np.random.default_rng(8)
    H, KV, hd, page, L, keep = 8, 2, 64, 16, 90, 40
    host = Host(16, KV, page, hd, K.INT8, 16, True, 2)
    table = np.array([[5, 1, 9, 0, 3, 11]], np.int32)
    dst_table = np.array([[2, 7, 12, 4]], np.int32)
    x = rng.standard_normal((2, L + 1, KV, hd)).astype(np.float32)
    q = (rng.standard_normal((4, H, hd)) * 2).astype(np.float32)
    cache = host.gpu()
    cache.append(up(x[0, :L]), up(x[1, :L]), batch(table, [0, L], [L]))
    host.append(x[0, :L], x[1, :L], table, [0, L], [L])
    w = torch.zeros((1, KV, 96), device="cuda")
    cache.attend(up(q[:3]), batch(table, [0, 3], [L]), weights=w)
    w2 = torch.zeros((1, KV, 96), device="cuda")
    rows, lens = cache.evict(w, batch(table, [0, 0], [L], max_q=1), up(dst_table), keep, 2, 8, weights_out=w2)
    wn = w.cpu().numpy()
    for h in range(KV):
        r = select_reference(wn[0, h], L, keep, 2, 8)
        assert (rows[0, h].cpu().numpy() == r).all()
        assert (w2[0, h, :keep].cpu().numpy() == wn[0, h, r]).all()
    # the next token goes to row `keep`, at position L
    cache.append(up(x[0, L:]), up(x[1, L:]), batch(dst_table, [0, 1], [keep + 1], q_pos=[L]))
    b = batch(dst_table, [0, 1], [keep + 1], q_pos=[L])
    out = cache.attend(up(q[3:]), b, K.Score(window=70), weights=w2)
    mirror = Host(16, KV, page, hd, K.INT8, 16, True, 2)
    mirror.k, mirror.v = cache.k.view(torch.uint8).cpu().numpy(), cache.v.view(torch.uint8).cpu().numpy()
    mirror.ks, mirror.vs, mirror.pos = cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy(), cache.pos.cpu().numpy()
    assert (mirror.pos[dst_table[0, keep // page], :, keep % page] == L).all()
    want, _, _, ds, mag, _ = reference(mirror, q[3:], dst_table, [0, 1], [keep + 1], H, window=70, q_pos=[L])
    assert_close(out.cpu().numpy(), want, out_bound(want, mag, ds, torch.float32))
