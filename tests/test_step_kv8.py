"""The decoder step on an 8-bit KV cache (tlmg_step_open with kv_dt
TLMG_DT_KV8_INT8 or _E4M3): the step's own projections, qk-norm and RoPE, then
append and attention on the layer's 8-bit rows.

Two layers, all-zero experts, and the output projection of one of the layers
zero: the K and V rows of both layers are then the oracle's bit for bit, so
their codes are too, and the logits differ from a 64-bit evaluation only by the
live layer's attention and by f32 sums. With b the attention's bound
(tests/test_kv8.py), O its output projection, h the residual, x = h r w the
normalised one and r = 1 / rms(h): |dh| <= |O| b + 2^-24 (n |O| |att| + 2 |h|),
n = H hd, and |dlogit| <= |head| (|w| r |dh| + |x| |dh|_2 / |h|_2) + 2^-24
(D + 8) |head| |x|; 1.01 covers the second order.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from conftest import same_bits
from test_kv8 import Host, out_bound, reference
from test_step import EPS, SHAPES, _model, _mv

from tierlm_b200 import _lib
from tierlm_b200 import kvcache as K

pytestmark = pytest.mark.gpu

KV_DT = {K.INT8: _lib.KV8_INT8, K.E4M3: _lib.KV8_E4M3}


def build(seed, shape, live):
    """_model with f32 output projections (zero but in layer `live`), an f32 lm_head and zero experts."""
    m = _model(seed, shape)
    c = dict(m["cfg"], HEAD_DT=0)
    rng = np.random.default_rng(seed + 1)
    D, n = c["D"], c["H"] * c["HD"]
    for l, A in enumerate(m["layers"]):
        o = (rng.standard_normal((D, n)) / math.sqrt(n)).astype(np.float32) if l == live else np.zeros((D, n), np.float32)
        A["o"] = o
        A["mats"][3] = o.view(np.uint8)
        A["dts"] = (*A["dts"][:3], 0)
        A["experts"] = [(np.zeros_like(p), off, dts) for p, off, dts in A["experts"]]
    m["head_f"] = (rng.standard_normal((c["V"], D)) / math.sqrt(D)).astype(np.float32)
    return dict(m, cfg=c, head=m["head_f"].view(np.uint8))


def context(m, fmt, max_ctx):
    from tierlm_b200.moe import MoeContext
    c = m["cfg"]
    ctx = MoeContext(len(m["layers"]), c["D"], c["DE"], c["E"], c["K"], router=0)
    for l, A in enumerate(m["layers"]):
        for e, (payload, off, dts) in enumerate(A["experts"]):
            ctx.set_expert(l, e, dts, payload, off)
        ctx.set_layer(l, ffn_norm=A["ffn_norm"], router_dt=0, router_w=A["router_w"], router_row_bytes=4 * c["D"])
    ctx.step_open(c["H"], c["KVH"], c["HD"], c["V"], m["inv"], 1.0, max_ctx=max_ctx, kv_dtype=KV_DT[fmt], attn_mode=1)
    for l, A in enumerate(m["layers"]):
        ctx.set_attention(l, A["attn_norm"], A["dts"], *A["mats"], q_norm=A["q_norm"], k_norm=A["k_norm"])
    ctx.set_embedding(c["EMB_DT"], m["emb"])
    ctx.set_output(m["out_norm"], c["HEAD_DT"], m["head"])
    return ctx


def expected(orc, m, fmt, live, tokens):
    """Logits of every position and their bounds."""
    c = m["cfg"]
    D, H, KVH, HD = (c[x] for x in ("D", "H", "KVH", "HD"))
    A = m["layers"][live]
    host = Host(1, KVH, 64, HD, fmt, 16)
    table = np.zeros((1, 1), np.int32)
    heads = lambda x, n: x.reshape(n, HD)  # noqa: E731
    logits, bounds = [], []
    for pos, tok in enumerate(tokens):
        h = orc.dequantize_row(c["EMB_DT"], m["emb"][tok], D)
        cs = np.array([np.float32(math.cos(pos * float(f))) for f in m["inv"]], np.float32)
        sn = np.array([np.float32(math.sin(pos * float(f))) for f in m["inv"]], np.float32)
        xb = orc.rmsnorm(h, A["attn_norm"], EPS)
        q = heads(_mv(orc, A["dts"][0], A["mats"][0], xb, H * HD), H)
        k = heads(_mv(orc, A["dts"][1], A["mats"][1], xb, KVH * HD), KVH)
        v = heads(_mv(orc, A["dts"][2], A["mats"][2], xb, KVH * HD), KVH)
        if A["q_norm"] is not None:
            q = np.stack([orc.rmsnorm(q[i], A["q_norm"], EPS) for i in range(H)])
            k = np.stack([orc.rmsnorm(k[i], A["k_norm"], EPS) for i in range(KVH)])

        def rope(x):
            a, b = x[:, : HD // 2], x[:, HD // 2:]
            return np.concatenate([a * cs - b * sn, b * cs + a * sn], axis=1).astype(np.float32)

        host.append(rope(k)[None], v[None], table, [0, 1], [pos + 1])
        att, _, _, ds, mags, _ = reference(host, rope(q)[None], table, [0, 1], [pos + 1], H)
        b = out_bound(att, mags, ds, torch.float32).reshape(-1)
        att = att.reshape(-1)
        O, w, head = A["o"].astype(np.float64), m["out_norm"].astype(np.float64), m["head_f"].astype(np.float64)
        y = h.astype(np.float64) + O @ att
        dy = np.abs(O) @ b + 2.0 ** -24 * (att.size * (np.abs(O) @ np.abs(att)) + 2 * np.abs(y))
        r = 1 / math.sqrt((y * y).mean() + EPS)
        x = y * r * w
        logits.append(head @ x)
        bounds.append(1.01 * (np.abs(head) @ (np.abs(w) * r * dy + np.abs(x) * np.linalg.norm(dy) / np.linalg.norm(y)) +
                              2.0 ** -24 * (D + 8) * (np.abs(head) @ np.abs(x))))
    return np.stack(logits), np.stack(bounds)


def run(ctx, tokens, V):
    out = np.zeros((len(tokens), V), np.float32)
    for pos, tok in enumerate(tokens):
        ctx.decode_step(tok, pos, out[pos])
    ctx.check()
    return out


@pytest.mark.parametrize("live", [0, 1])
@pytest.mark.parametrize("fmt", [K.INT8, K.E4M3])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_step_kv8(orc, shape, fmt, live):
    """Every position's logits, past a scale block (16) and a tile of rows
    (32); a second run over the same positions and eager steps give the
    same bits."""
    _lib.check(_lib.load().tlmg_init(0))
    m = build(11, shape, live)
    V = m["cfg"]["V"]
    tokens = [int(t) for t in np.random.default_rng(3).integers(0, V, 37)]
    ctx = context(m, fmt, 41)
    got = run(ctx, tokens, V)
    again = run(ctx, tokens, V)
    assert ctx.step_info()["replays"] > 0
    ctx.step_graphs(False)
    eager = run(ctx, tokens, V)
    ctx.close()
    want, bound = expected(orc, m, fmt, live, tokens)
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    assert same_bits(again, got).all() and same_bits(eager, got).all()


def test_step_kv8_one_position(orc):
    """max_ctx 1: one page of one tile."""
    _lib.check(_lib.load().tlmg_init(0))
    m = build(12, "small", 0)
    ctx = context(m, K.INT8, 1)
    got = run(ctx, [5], m["cfg"]["V"])
    with pytest.raises(_lib.TlmError) as ei:
        ctx.decode_step(5, 1, got[0])
    assert ei.value.code == _lib.TLMG_ERANGE
    ctx.close()
    want, bound = expected(orc, m, K.INT8, 0, [5])
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("kv_dtype,mode", [(_lib.KV8_INT8, 0), (_lib.KV8_E4M3, 0), (0x100, 1), (0x103, 1)])
def test_step_kv8_refusals(kv_dtype, mode):
    """The exact mode has no 8-bit form, and there are two formats."""
    from tierlm_b200.moe import MoeContext
    _lib.check(_lib.load().tlmg_init(0))
    m = _model(6)
    c = m["cfg"]
    ctx = MoeContext(len(m["layers"]), c["D"], c["DE"], c["E"], c["K"], router=0)
    with pytest.raises(_lib.TlmError) as ei:
        ctx.step_open(c["H"], c["KVH"], c["HD"], c["V"], m["inv"], 1.0, max_ctx=16, kv_dtype=kv_dtype, attn_mode=mode)
    assert ei.value.code == _lib.TLMG_EINVAL
    ctx.close()
