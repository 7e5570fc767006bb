"""Edges of the 8-bit KV cache (tierlm_b200/kvcache.py) beside tests/test_kv8.py, whose restatement and bounds it uses."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_kv8 import WIDE, Host, assert_cache, batch, check_attend, make, quantise, select_reference, tables, up

from tierlm_b200 import kvcache as K


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
