"""Edges of the 8-bit KV cache (tierlm_b200/kvcache.py) beside tests/test_kv8.py, whose restatement and bounds it uses."""
from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest
import torch

from test_kv8 import WIDE, Host, assert_cache, batch, c_batch, c_cache, c_score, check_attend, make, quantise, select_reference, tables, up

from tierlm_b200 import _lib
from tierlm_b200 import kvcache as K


# ---- bounds of zero ----------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(max_q=0), dict(total_q=0), dict(total_q=0, max_q=0), dict(max_kv=0), dict(max_q=0, max_kv=0)])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("weights", [0, 1])
def test_work_bytes_of_empty_calls(kw, hd, weights):
    L = _lib.load()
    got = L.tlmg_kv8_attend_work_bytes(C.byref(c_cache(hd=hd)), C.byref(c_batch(**kw)), C.byref(c_score()), 4, 0, weights)
    assert 0 < got < 1 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bounds_of_zero(dtype):
    """Tokens where max_q allows none: NaN, and weights as they were."""
    lens, news, H, KV, hd = [20, 30], [2, 1], 4, 2, 64
    host, table, q_start, q, _ = make(43, lens, news, H, KV, hd, dtype=dtype)
    cache = host.gpu()
    for bounds in (dict(max_q=0), dict(max_q=0, max_kv=0)):
        w = torch.full((2, KV, 33), 0.5, device="cuda")
        out, lse = cache.attend(q.cuda(), batch(table, q_start, lens, **bounds), lse=True, weights=w)
        assert torch.isnan(out).all() and torch.isnan(lse).all() and (w == 0.5).all()
    out, lse = cache.attend(q[:0].cuda(), batch(table, [0, 0, 0], lens), lse=True)
    assert out.shape == (0, H, hd) and lse.shape == (0, H)
    out = cache.attend(q[:0].cuda(), batch(table, [0, 0, 0], [0, 0]))
    assert out.shape == (0, H, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_without_rows(dtype):
    """max_kv 0: tokens have no row of their own, so they are NaN; sequences without tokens are in order. Weights stay."""
    lens, news, H, KV, hd = [20, 30], [2, 1], 4, 2, 64
    host, table, q_start, q, _ = make(43, lens, news, H, KV, hd, dtype=dtype)
    cache = host.gpu()
    w = torch.full((2, KV, 33), 0.5, device="cuda")
    out, lse = cache.attend(q.cuda(), batch(table, q_start, lens, max_kv=0), lse=True, weights=w)
    assert torch.isnan(out).all() and torch.isnan(lse).all() and (w == 0.5).all()
    none = torch.empty((2, KV, 0), device="cuda")
    out = cache.attend(q[:0].cuda(), batch(table, [0, 0, 0], [0, 0]), weights=none)
    assert out.shape == (0, H, hd)



# ---- calls from several threads -----------------------------------------------------------
def test_score_struct_lives_as_long_as_the_score():
    """Calls with other batch sizes and head counts leave the struct where it is: a call of another thread may be reading it."""
    s = K.Score(softcap=5.0, window=7)
    at = s._at(1, 8, 0)
    assert all(s._at(n, H, 0) == at for n in range(1, 50) for H in (8, 16, 32))
    c = K._Score.from_address(at)
    assert (c.softcap, c.window, c.causal, c.doc_stride, c.slopes) == (5.0, 7, 1, 0, None)


def test_batch_struct_per_number_of_tokens():
    """A call on other numbers of tokens leaves the struct of an earlier one as it was."""
    b = K.Kv8Batch.__new__(K.Kv8Batch)
    b.q_pos, b._dev, b._calls, b._c = None, 0, {}, c_batch(total_q=0, max_q=9, max_kv=50)
    at = [b._at(n, 0) for n in range(20)]
    assert len(set(at)) == 20 and [b._at(n, 0) for n in range(20)] == at
    for n, p in enumerate(at):
        c = K._Batch.from_address(p)
        assert (c.total_q, c.max_q, c.max_kv, c.n_seq) == (n, 9, 50, 2)


@pytest.mark.gpu
def test_threads():
    """Threads with streams of their own share a cache, the default score and a batch; every call has its own sizes."""
    lens, H, KV, hd = [300, 200, 100], 4, 2, 64
    host, table, _, _, rng = make(44, lens, [0, 0, 0], H, KV, hd)
    cache = host.gpu()
    shared = batch(table, [0, 1, 2, 3], lens)
    q = up(rng.standard_normal((8, 16, hd)).astype(np.float32))
    jobs = []
    for i in range(4):
        n = 1 + i % 3
        own = batch(table[:n], list(range(n + 1)), lens[:n])
        jobs += [(own, q[:n, :2 * (i + 1)].contiguous()), (shared, q[:3 + i, :4].contiguous())]
    want = [cache.attend(x, b)[:b.n_seq].clone() for b, x in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(400):
                j = (i * (2 * k + 1) + k) % len(jobs)
                b, x = jobs[j]
                if not torch.equal(cache.attend(x, b)[:b.n_seq], want[j]):
                    wrong.append((k, i, j))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong, wrong[:5]



@pytest.mark.gpu
def test_threads_on_one_stream():
    """Calls of several kernels from threads on the same stream: each joins its own partial results."""
    lens, H, KV, hd = [3000, 1800], 8, 2, 64
    host, table, _, _, rng = make(45, lens, [0, 0], H, KV, hd, page=64)
    caches = [host.gpu() for _ in range(2)]
    q = up(rng.standard_normal((4, H, hd)).astype(np.float32))
    jobs = [(batch(table[:1], [0, 1 + i], lens[:1]), q[:1 + i]) for i in range(4)] + [(batch(table, [0, 1, 3], lens), q[:3])]
    want = [caches[0].attend(x, b) for b, x in jobs]
    torch.cuda.synchronize()
    got = {}

    def work(k):
        for i in range(300):
            j = (i * (2 * k + 1) + k) % len(jobs)
            got[k, i] = j, caches[k % 2].attend(jobs[j][1], jobs[j][0])

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert len(got) == 1200 and all(torch.equal(out, want[j]) for j, out in got.values())


# ---- devices ------------------------------------------------------------------------------
@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_refuses_tensors_of_other_devices(monkeypatch):
    """Everything a call reads has to be on the cache's device, and that the current one: no call reaches the library."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    def called(*a):
        raise AssertionError("the library was called")

    def refused(fn, what):
        with pytest.raises(_lib.TlmError) as e:
            fn()
        assert e.value.code == -3 and "cuda:" in str(e.value) and what in str(e.value), str(e.value)

    monkeypatch.setattr(K, "_current_device", lambda: 0, raising=False)
    monkeypatch.setattr(K, "_raw_stream", lambda index: 0)
    i32 = lambda d, *shape: torch.empty(shape, dtype=torch.int32, device=f"cuda:{d}")  # noqa: E731
    f32 = lambda d, *shape: torch.empty(shape, device=f"cuda:{d}")  # noqa: E731
    with FakeTensorMode():
        pools = lambda *d: (f32(d[0], 4, 2, 16, 64).to(torch.int8), f32(d[1], 4, 2, 16, 64).to(torch.int8),  # noqa: E731
                            f32(d[2], 4, 2, 1), f32(d[3], 4, 2, 1), i32(d[4], 4, 2, 16))
        for i, what in enumerate(["v", "k_scale", "v_scale", "pos"], 1):
            d = [0] * 5
            d[i] = 1
            refused(lambda: K.Kv8Cache.from_pools(*pools(*d)), what)
        cache, other = K.Kv8Cache.from_pools(*pools(*[0] * 5)), K.Kv8Cache.from_pools(*pools(*[1] * 5))
        for c in (cache, other):
            c._append = c._read = c._attend = c._need = c._select = c._compact = called
        arrays = lambda *d: (i32(d[0], 3, 2), i32(d[1], 4), i32(d[2], 3), 1, 20, i32(d[3], 3))  # noqa: E731
        for i, what in enumerate(["q_start", "kv_len", "q_pos"], 1):
            d = [0] * 4
            d[i] = 1
            refused(lambda: K.Kv8Batch(*arrays(*d)), what)
        b, far = K.Kv8Batch(*arrays(*[0] * 4)), K.Kv8Batch(*arrays(*[1] * 4))
        rows, q, w, table = f32(0, 3, 2, 64), f32(0, 3, 4, 64), f32(0, 3, 2, 20), i32(0, 3, 2)
        refused(lambda: cache.append(f32(1, 3, 2, 64), rows, b), "k ")
        refused(lambda: cache.append(rows, f32(1, 3, 2, 64), b), "v ")
        refused(lambda: cache.append(rows, rows, far), "batch")
        refused(lambda: cache.attend(f32(1, 3, 4, 64), b), "q ")
        refused(lambda: cache.attend(q, far), "batch")
        refused(lambda: cache.attend(q, b, out=f32(1, 3, 4, 64)), "out")
        refused(lambda: cache.attend(q, b, lse=f32(1, 3, 4)), "lse")
        refused(lambda: cache.attend(q, b, weights=f32(1, 3, 2, 20)), "weights")
        for kw in (dict(slopes=f32(1, 4)), dict(prefix=i32(1, 3)), dict(doc=i32(1, 3, 20))):
            refused(lambda: cache.attend(q, b, K.Score(**kw)), next(iter(kw)))
        row0, start = i32(0, 3), i32(0, 4)
        refused(lambda: cache.read(i32(1, 3, 2), row0, start, 5), "page_table")
        refused(lambda: cache.read(table, i32(1, 3), start, 5), "row0")
        refused(lambda: cache.read(table, row0, i32(1, 4), 5), "start")
        refused(lambda: cache.read(table, row0, start, 5, k=f32(1, 5, 2, 64), v=f32(0, 5, 2, 64)), "k ")
        refused(lambda: cache.evict(f32(1, 3, 2, 20), b, table, 8), "weights")
        refused(lambda: cache.evict(w, far, table, 8), "batch")
        refused(lambda: cache.evict(w, b, table, 8, dst=other), "destination")
        refused(lambda: cache.evict(w, b, table, 8, rows=i32(1, 3, 2, 8)), "rows")
        refused(lambda: cache.evict(w, b, table, 8, lens=i32(1, 3)), "lens")
        refused(lambda: cache.evict(w, b, i32(1, 3, 2), 8), "dst_table")
        refused(lambda: cache.evict(w, b, table, 8, weights_out=f32(1, 3, 2, 8)), "weights_out")
        # all of it on another device than the current one
        refused(lambda: other.append(f32(1, 3, 2, 64), f32(1, 3, 2, 64), far), "current device")
        refused(lambda: other.attend(f32(1, 3, 4, 64), far), "current device")
        refused(lambda: other.read(i32(1, 3, 2), i32(1, 3), i32(1, 4), 5), "current device")
        refused(lambda: other.evict(f32(1, 3, 2, 20), far, i32(1, 3, 2), 8), "current device")


# ---- scratch ------------------------------------------------------------------------------
@pytest.mark.gpu
def test_scratch_is_shared_and_bounded():
    """Layers used on one stream take one scratch; that of a prompt is torch's again after the call."""
    KV, hd, page, L, n = 2, 128, 64, 20000, 2000
    caches = [K.Kv8Cache(-(-L // page), KV, page, hd) for _ in range(3)]
    table = torch.arange(-(-L // page), dtype=torch.int32, device="cuda")[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    one, many = K.Kv8Batch(table, i32(0, 1), i32(L), 1, L), K.Kv8Batch(table, i32(0, n), i32(L), n, L)
    q = torch.randn((n, 32, hd), device="cuda").to(torch.bfloat16)
    out, few = torch.empty_like(q), torch.empty_like(q[:1])
    caches[0].attend(q[:1], one, out=few)
    at = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()      # (earlier tests' peak is not these calls')
    for c in caches:
        c.attend(q[:1], one, out=few)
        c.attend(q, many, out=out)
    assert torch.cuda.memory_allocated() == at
    peak = torch.cuda.max_memory_allocated()
    assert peak - at < 1 << 30


@pytest.mark.gpu
@pytest.mark.parametrize("news,H", [([1, 1], 8), ([40, 30], 16)])
def test_graph_replay_after_larger_calls(news, H):
    """A captured call's scratch stays its own: larger calls on the capture's stream and new tensors between the replays
    neither change its output nor are changed by it."""
    lens, KV, hd = [3000, 1700], 2, 64
    host, table, q_start, q, rng = make(46, lens, news, H, KV, hd, page=64)
    cache, b, qd = host.gpu(), batch(table, q_start, lens), q.cuda()
    more = [0, 60, 120]
    large, ql = batch(table, more, lens), up(rng.standard_normal((120, H, hd)).astype(np.float32))
    w, wl = (torch.zeros((2, KV, 3000), device="cuda") for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = cache.attend(qd, b, weights=w).clone()
        for _ in range(2):
            cache.attend(qd, b, weights=w)
    torch.cuda.synchronize()
    w.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = cache.attend(qd, b, weights=w)
    with torch.cuda.stream(s):
        first = cache.attend(ql, large, weights=wl).clone()
        fills = [torch.full((1 << 18,), float(i), device="cuda") for i in range(64)]
    torch.cuda.synchronize()
    for i in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all((f == i).all() for i, f in enumerate(fills))
    with torch.cuda.stream(s):
        assert torch.equal(cache.attend(ql, large, weights=wl), first)
    one = torch.zeros_like(w)
    cache.attend(qd, b, weights=one)
    torch.testing.assert_close(w, 3 * one, rtol=2.0 ** -20, atol=0)


# ---- eviction ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("src_fmt,dst_fmt", [(K.INT8, K.INT8), (K.E4M3, K.INT8), (K.INT8, K.E4M3)])
@pytest.mark.parametrize("keep", [33, 40, 64, 100, 161])
@pytest.mark.parametrize("hd,dblock", [(64, 32), (64, 64), (64, 128), (64, 256), (128, 64), (256, 128)])
def test_evict_large_blocks(hd, dblock, keep, src_fmt, dst_fmt):
    """Destination blocks of more rows than a warp has lanes, whole and in part; chosen rows on a bad page, among the last
    of a block too, are left out."""
    rng = np.random.default_rng(41)
    lens, KV, page, block, dpage = [300, 170, 45], 2, 16, 4, 256
    host, table, _, _, _ = make(42, lens, [0, 0, 0], 2, KV, hd, src_fmt, page, block, True)
    bad = table.copy()
    bad[0, 1], bad[0, 12], bad[1, 7], bad[2, 2] = -1, 1 << 20, host.k.shape[0], -7
    w = rng.random((3, KV, 300)).astype(np.float32)
    dtable, n_dst = tables(rng, [min(L, keep) for L in lens], dpage)
    dst = Host(n_dst, KV, dpage, hd, dst_fmt, dblock, True, 9)
    src_gpu, dst_gpu = host.gpu(), dst.gpu()
    w_out = torch.full((3, KV, keep), 7.0, device="cuda")
    rows, _ = src_gpu.evict(up(w), batch(bad, [0, 0, 0, 0], lens, max_q=1), up(dtable), keep, 3, 9, dst=dst_gpu, weights_out=w_out)
    want_w = np.zeros((3, KV, keep), np.float32)
    for s, L in enumerate(lens):
        kr, vr, pr = host.rows("k", table[s], L), host.rows("v", table[s], L), host.positions(table[s], L)
        ok = np.array([0 <= bad[s, t // page] < host.k.shape[0] for t in range(L)])
        for h in range(KV):
            r = select_reference(w[s, h], L, keep, 3, 9)
            assert (rows[s, h].cpu().numpy()[:len(r)] == r).all()
            want_w[s, h, :len(r)] = np.where(ok[r], w[s, h, r], 0)
            for j0 in range(0, len(r), dblock):
                rr = r[j0:j0 + dblock]
                have = ok[rr]
                at = np.nonzero(have)[0]
                if at.size == 0:
                    continue
                e, o = dtable[s, j0 // dpage], j0 % dpage
                for x, codes, scale in ((kr, dst.k, dst.ks), (vr, dst.v, dst.vs)):
                    c, d = quantise(x[rr[at], h].astype(np.float32), dst_fmt)
                    codes[e, h, o + at], scale[e, h, o // dblock] = c, d
                dst.pos[e, h, o + at] = pr[rr[at], h]
    assert_cache(dst_gpu, dst)
    assert (w_out.cpu().numpy() == want_w).all()


@pytest.mark.gpu
def test_compact_rows_past_the_weights():
    """Rows of the caller's own choice that have no weight: they move, their weight is 0."""
    L, KV, page, n_keep, stride = 100, 2, 16, 12, 40
    host, table, _, _, rng = make(47, [L], [0], 2, KV, 64, K.INT8, page, 16, True)
    src, dst = host.gpu(), Host(2, KV, page, 64, K.INT8, 16, True, 3).gpu()
    r = np.stack([np.sort(rng.permutation(L)[:n_keep]) for _ in range(KV)])[None].astype(np.int32)
    r[0, 0, :3], r[0, 1, -3:] = [38, 39, 40], [98, 99, -1]
    r[0, 0] = np.sort(r[0, 0])
    w = rng.random((1, KV, stride)).astype(np.float32)
    wd, rd, td, ld, dd = up(w), up(r), up(table), up(np.array([L], np.int32)), up(np.array([[1]], np.int32))
    out = torch.full((1, KV, n_keep), 7.0, device="cuda")
    _lib.check(_lib.load().tlmg_kv8_compact(src._p, dst._p, 1, td.data_ptr(), td.shape[1], ld.data_ptr(), dd.data_ptr(), 1, rd.data_ptr(),
                                            n_keep, wd.data_ptr(), stride, out.data_ptr(), n_keep, 1))
    want = np.where((r >= 0) & (r < stride), np.take_along_axis(w, np.clip(r, 0, stride - 1), 2), 0)
    assert (out.cpu().numpy() == want).all()
    assert (dst.pos[1].cpu().numpy()[:, :n_keep][r[0] >= 0] == host.positions(table[0], L)[r[0], np.arange(KV)[:, None]][r[0] >= 0]).all()


@pytest.mark.parametrize("at", [0, 4, -4, 4 * (2 * 2 * 40) - 4, -4 * (2 * 2 * 12) + 4])
def test_weights_out_over_weights(at):
    """Kept weights may not go where the weights are read from, in part neither."""
    L, ok, w = _lib.load(), 1 << 20, 1 << 24
    rc = L.tlmg_kv8_compact(C.byref(c_cache()), C.byref(c_cache()), 2, ok, 4, ok, ok, 4, ok, 8, w, 40, w + at, 12, 1)
    assert rc == -3 and b"overlaps" in L.tlmg_errmsg()


@pytest.mark.gpu
def test_weights_out_beside_weights():
    """The buffer right behind the weights is another one; entries from n_keep on stay as they were."""
    L, KV, keep = 60, 2, 20
    host, table, _, _, rng = make(48, [L], [0], 2, KV, 64, K.INT8, 16, 16, True)
    both = torch.full((2 * KV * L,), 7.0, device="cuda")
    w, out = both[:KV * L].view(1, KV, L), both[KV * L:].view(1, KV, L)
    wn = rng.random((1, KV, L)).astype(np.float32)
    w.copy_(up(wn))
    rows, _ = host.gpu().evict(w, batch(table, [0, 0], [L], max_q=1), up(np.array([[0, 1]], np.int32)), keep, 2, 4,
                               dst=Host(2, KV, 16, 64, K.INT8, 16, True, 3).gpu(), weights_out=out)
    assert (out[..., :keep].cpu().numpy() == np.take_along_axis(wn, rows.cpu().numpy(), 2)).all() and (out[..., keep:] == 7.0).all()


# ---- attention ----------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
def test_wide_rising_scores(hd, dtype):
    """Scores that rise from key tile to key tile, now in the one and now in the other half of a tile: every tile moves the
    reference that the two threads of a query row agree on."""
    rng = np.random.default_rng(51)
    L, n, H, KV, page = 1700, 90, 4, 2, 64
    table, n_pages = tables(rng, [L], page)
    host = Host(n_pages, KV, page, hd, K.INT8, 16)
    u = rng.standard_normal(hd) / np.sqrt(hd)
    t = np.arange(L)
    rise = 3.0 * (t // 128) + np.where((t // 64 + t // 128) % 2 == 0, 2.0, 0.0)
    k = (rng.standard_normal((L, KV, hd)) * 0.3 + (rise[:, None] * u)[:, None]).astype(np.float32)
    host.append(k, rng.standard_normal((L, KV, hd)).astype(np.float32), table, [0, L], [L])
    q = torch.from_numpy(((rng.standard_normal((n, H, hd)) * 0.3 + u * rng.uniform(0.5, 2, (n, H, 1)) * np.sqrt(hd))).astype(np.float32)).to(dtype)
    for causal in (True, False):
        check_attend(host, table, [0, n], [L], q, H, max_kv=WIDE, causal=causal)


def on_device(cache, table_row, L, q, H, scale=0.0, visible=None):
    """64-bit attention of q [n][H][hd] over rows 0 .. L - 1 of one sequence, on the GPU: out, sum p |v|, sum |q k| scale at
    its largest; visible [n] rows (None: all L)."""
    row0 = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = cache.read(table_row[None].contiguous(), row0, torch.tensor([0, L], dtype=torch.int32, device="cuda"), L)
    n, hd, KV = q.shape[0], q.shape[2], k.shape[1]
    scale = scale or hd ** -0.5
    out, mag = (torch.empty((n, H, hd), dtype=torch.float64, device="cuda") for _ in range(2))
    top = torch.empty((n, H), dtype=torch.float64, device="cuda")
    for h in range(H):
        kk, vv = k[:, h * KV // H].double(), v[:, h * KV // H].double()
        z = scale * (q[:, h].double() @ kk.T)
        size = scale * (q[:, h].double().abs() @ kk.abs().T)
        if visible is not None:
            hidden = torch.arange(L, device="cuda")[None] >= visible[:, None]
            z, size = z.masked_fill(hidden, -torch.inf), size.masked_fill(hidden, 0)
        p = torch.softmax(z, -1)
        out[:, h], mag[:, h], top[:, h] = p @ vv, p @ vv.abs(), size.amax(-1)
    return out, mag, top


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,n_seq,T", [(64, 1, 2368), (128, 1, 2368), (64, 74, 32)])
def test_long_rows(hd, n_seq, T, dtype):
    """131,072 rows of positive values under even weights, in as many items as the SMs take whole (their key tiles stay one
    sum), on images (1 sequence) and with converting warps (74 over the same pages). Each output: the bounds of test_kv8.py
    and 2^-13 sum p |v| for the tensor core's sums, which truncate by 2^-23 of it at most, 1,024 times a run of 128 key tiles.
    f16's mean relative error over all of these outputs: 2^-13 from the runs and 2^-14 for the mean of the roundings, uniform in 2^-12
    at most over columns of different size. (One run over all rows: 8e-4.)"""
    L, H, KV, page = 131072, 16, 1, 128
    g = torch.Generator(device="cuda").manual_seed(hd)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    cache = K.Kv8Cache(L // page, KV, page, hd)
    table = torch.randperm(L // page, generator=g, device="cuda").to(torch.int32)
    v = (0.5 + torch.rand((1, KV, hd), generator=g, device="cuda")) * (1 + 0.25 * torch.rand((L, KV, hd), generator=g, device="cuda"))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache.append(rnd(L, KV, hd), v, K.Kv8Batch(table[None].contiguous(), i32(0, L), i32(L), L, L))
    q = (rnd(n_seq * T, H, hd) * 0.2).to(dtype)
    b = K.Kv8Batch(table[None].repeat(n_seq, 1), torch.arange(n_seq + 1, dtype=torch.int32, device="cuda") * T,
                   torch.full((n_seq,), L, dtype=torch.int32, device="cuda"), T, L)
    got = cache.attend(q, b, K.Score(causal=False))
    at = torch.cat([torch.arange(12), torch.arange(n_seq * T - 12, n_seq * T)]).cuda()
    want, mag, top = on_device(cache, table, L, q[at], H)
    out = got[at].double()
    bound = (2.0 ** -18 * top[..., None] + 2.0 ** -18) * mag + 1e-11
    if dtype != torch.float32:
        # one f16 a weight, the truncated sums, the output (f16's smallest step comes to less than 1e-11 here)
        bound = 1.01 * (bound + 2.0 ** -11 * mag + 2.0 ** -13 * mag) + want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11)
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() / bound).max())
    if dtype == torch.float16:
        mean = float(((out - want) / want).mean())
        assert abs(mean) <= 2.0 ** -13 + 2.0 ** -14, mean


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("hd,KV,H", [(256, 2, 32), (256, 8, 16), (128, 2, 32), (64, 4, 64), (256, 1, 16)])
@pytest.mark.parametrize("n", [16384, 1 << 20])
def test_long_prompts_are_served(hd, KV, H, n, dt):
    """No number of tokens whose rows of all heads can be counted is refused."""
    L = _lib.load()
    b = c_batch(n_seq=1, total_q=n, max_q=n, max_kv=n, table_stride=n // 16)
    assert L.tlmg_kv8_attend_work_bytes(C.byref(c_cache(hd=hd, KV=KV)), C.byref(b), C.byref(c_score()), H, dt, 0) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [256, 64])
def test_long_prompt_against_64_bits(hd, dtype):
    """A prompt of 16,500 tokens of 32 heads: first, middle and last tokens, and a sequence of too many tokens beside it
    (head_dim 256, f32: more query tiles than a grid's second dimension takes). Bounds of test_kv8.py; f16's smallest step comes to
    less than 2^-39 * 127 * 16,500 * the largest scale of V."""
    L, H, KV, page = 16500, 32, 2, 64
    g = torch.Generator(device="cuda").manual_seed(hd)
    k, v, q = (torch.randn((L + 3, h, hd), generator=g, device="cuda").to(dtype) for h in (KV, KV, H))
    cache = K.Kv8Cache(-(-L // page) + 1, KV, page, hd)
    table = torch.randperm(-(-L // page) + 1, generator=g, device="cuda").to(torch.int32)[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    one = K.Kv8Batch(table, i32(0, L), i32(L), L, L)
    cache.append(k[:L], v[:L], one)
    b = K.Kv8Batch(table.repeat(2, 1), i32(0, L, L + 3), i32(L, 2), L, L)
    got, lse = cache.attend(q, b, lse=True)
    assert torch.isnan(got[L:]).all() and torch.isnan(lse[L:]).all() and torch.isfinite(got[:L]).all()
    at = torch.tensor([0, 1, 2, 63, 64, 127, 128, 8190, 8191, 8192, 8193, 16374, 16375, 16376, 16384, L - 2, L - 1], device="cuda")
    want, mag, top = on_device(cache, table[0], L, q[at], H, visible=at + 1)
    low = 2.0 ** -39 * 127 * L * float(cache.v_scale.max())
    bound = (2.0 ** -18 * top[..., None] + 2.0 ** -18) * mag + 2.0 ** -11 * low
    if dtype == torch.bfloat16:
        bound = 1.01 * (bound + 2.0 ** -11 * mag + 2.0 ** -13 * mag + low) + want.abs() * 2.0 ** -8
    out = got[at].double()
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() / bound).max())
