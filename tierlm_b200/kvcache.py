"""The 8-bit KV cache on CUDA tensors: append, attention, eviction (the
tlmg_kv8_* calls of include/tlmg.h; no counterpart in the reference, whose KV
is f32).

One layer's K and V rows are 8-bit codes in page pools [n_pages][KV][page]
[hd] (torch.int8, or torch.float8_e4m3fn) with one f32 scale per `block` rows
of a head. A batch of sequences shares the pools: `Kv8Batch` holds the page
tables, the lengths and where each sequence's new tokens sit. Calls run on
torch's current stream. Scratch of up to KEEP bytes is kept for each stream,
for all caches (the layers of a model) that are used on it; what is larger, and
all scratch of a call under graph capture, is torch's for the call.
"""
from __future__ import annotations

import ctypes as C
import threading
from dataclasses import dataclass

import torch

from ._lib import BF16, F16, F32, TLMG_ERANGE, TlmError, check, load
from .quant import CUDA_STREAM_LEGACY, _dev

INT8, E4M3 = 1, 2
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream(index: int) -> int:
    """The current stream of a device for the C calls (see quant.stream_handle; without building a Stream object). It has
    to be the current device, on which the library launches: kernels elsewhere could not read the pools."""
    if _current_device() != index:
        raise TlmError(-3, f"the cache is on cuda:{index}, the current device is cuda:{_current_device()}")
    s = _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream
    return s if s else CUDA_STREAM_LEGACY


# A call's scratch up to this size is kept: torch.empty takes 1.8 us, a call from Python on 701 rows 17. Prompts take up to
# 600 MB, in calls that are long beside it.
KEEP = 32 << 20
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


class _Scratch:
    """What is kept for a stream. The lock covers a call's launches: those of two threads on one stream must not mix, since
    the later kernels of a call read what the first one left here. It may grow, never under capture: an outgrown buffer
    goes back to torch, which gives it to later work of the same stream."""
    __slots__ = ("lock", "size", "at", "buffer")

    def __init__(self, device):
        self.lock = threading.Lock()
        self.grow(1 << 20, device)

    def grow(self, size: int, device) -> None:
        self.buffer = torch.empty(size, dtype=torch.uint8, device=device)
        self.size, self.at = size, self.buffer.data_ptr()


_scratch: dict[tuple[int, int], _Scratch] = {}     # (device, stream)


_FMT = {torch.int8: INT8, torch.float8_e4m3fn: E4M3}
_X_DT = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class _Cache(C.Structure):
    """tlmg_kv8."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("pos", C.c_void_p), ("fmt", C.c_int32), ("n_pages", C.c_int32), ("KV", C.c_int32),
                ("page", C.c_int32), ("block", C.c_int32), ("hd", C.c_int32)]


class _Batch(C.Structure):
    """tlmg_kv8_batch."""
    _fields_ = [("page_table", C.c_void_p), ("q_start", C.c_void_p), ("kv_len", C.c_void_p), ("q_pos", C.c_void_p),
                ("n_seq", C.c_int32), ("table_stride", C.c_int32), ("total_q", C.c_int32), ("max_q", C.c_int32),
                ("max_kv", C.c_int32)]


class _Score(C.Structure):
    """tlmg_kv8_score."""
    _fields_ = [("scale", C.c_float), ("softcap", C.c_float), ("slopes", C.c_void_p), ("prefix", C.c_void_p),
                ("doc", C.c_void_p), ("doc_stride", C.c_int32), ("causal", C.c_int32), ("window", C.c_int32)]


def _ptr(t: torch.Tensor, what: str, dev: int) -> int:
    """The address of a contiguous tensor on CUDA device dev (calls of a few microseconds: one check does for "CUDA" and "which")."""
    if t.get_device() != dev:
        raise TlmError(-3, f"{what} is on {t.device}, not on cuda:{dev} as the rest")
    if not t.is_contiguous():
        raise TlmError(-3, f"{what} must be contiguous")
    return t.data_ptr()


def _i32(t: torch.Tensor | None, what: str, shape: tuple | None = None, dev: int | None = None) -> int | None:
    """The address of an int32 tensor of this shape on CUDA device dev (None: any)."""
    if t is None:
        return None
    if t.dtype != torch.int32:
        raise TlmError(-3, f"{what} must be int32, not {t.dtype}")
    if shape is not None and t.shape != shape:
        raise TlmError(-3, f"{what} has shape {tuple(t.shape)}, not {shape}")
    return _dev(t, what) if dev is None else _ptr(t, what, dev)


def _f32(t: torch.Tensor | None, what: str, shape: tuple | None = None, dev: int | None = None) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.float32:
        raise TlmError(-3, f"{what} must be float32, not {t.dtype}")
    if shape is not None and t.shape != shape:
        raise TlmError(-3, f"{what} has shape {tuple(t.shape)}, not {shape}")
    return _dev(t, what) if dev is None else _ptr(t, what, dev)


def _rows(t: torch.Tensor, what: str, heads: int, hd: int, dev: int) -> tuple[torch.Tensor, int, int]:
    """[n][heads][hd] rows, their stride in elements and their address; a copy
    where the library cannot read them in place (heads apart, rows off 16 bytes)."""
    if t.dtype not in _X_DT:
        raise TlmError(-3, f"{what} must be float32, float16 or bfloat16, not {t.dtype}")
    if t.dim() != 3 or t.shape[1:] != (heads, hd):
        raise TlmError(-3, f"{what} has shape {tuple(t.shape)}, not [n][{heads}][{hd}]")
    if t.get_device() != dev:
        raise TlmError(-3, f"{what} is on {t.device}, not on cuda:{dev} as the cache")
    st, sh, sd = t.stride()
    at = t.data_ptr()
    if sd != 1 or sh != hd or st < heads * hd or st * (4 if t.dtype is torch.float32 else 2) % 16 or at % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        st, at = heads * hd, t.data_ptr()
    return t, st, at


class Kv8Batch:
    """Sequences with new tokens: page_table int32 [n_seq][stride]; q_start
    int32 [n_seq + 1] (sequence s's new tokens are rows q_start[s] ..
    q_start[s + 1] - 1 of the token-major tensors); kv_len int32 [n_seq] rows
    per sequence, the new ones last; max_q and max_kv bound the two on the
    host; q_pos int32 [n] positions of the tokens (None: their row numbers)."""

    def __init__(self, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, max_q: int, max_kv: int,
                 q_pos: torch.Tensor | None = None):
        if page_table.dim() != 2:
            raise TlmError(-3, f"page_table has shape {tuple(page_table.shape)}, not [n_seq][stride]")
        n_seq, stride = page_table.shape
        self._keep = (page_table, q_start, kv_len, q_pos)
        self.n_seq, self.page_table, self.kv_len, self.q_pos = n_seq, page_table, kv_len, q_pos
        self.max_q, self.max_kv = max_q, max_kv
        self._dev = dev = page_table.get_device()
        self._c = _Batch(_i32(page_table, "page_table"), _i32(q_start, "q_start", (n_seq + 1,), dev),
                         _i32(kv_len, "kv_len", (n_seq,), dev), _i32(q_pos, "q_pos", None, dev), n_seq, stride, 0, max_q, max_kv)
        self._calls: dict[int, tuple[_Batch, int]] = {}     # tokens -> struct, address

    def _at(self, total: int, dev: int) -> int:
        """The address of the C struct for a call on `total` tokens and device dev: one for each number of tokens, as long as the batch
        lives (another thread's call may be reading it)."""
        if self._dev != dev:
            raise TlmError(-3, f"the batch is on cuda:{self._dev}, the cache on cuda:{dev}")
        made = self._calls.get(total)
        if made is None:
            if self.q_pos is not None and self.q_pos.numel() < total:
                raise TlmError(-3, f"q_pos has {self.q_pos.numel()} entries for {total} tokens")
            c = _Batch.from_buffer_copy(self._c)
            c.total_q = total
            made = self._calls.setdefault(total, (c, C.addressof(c)))
        return made[1]


@dataclass(frozen=True)
class Score:
    """How scores are formed and masked (tlmg_kv8_score): softcap c > 0:
    c * tanh(z / c); slopes f32 [H]: minus slopes[h] * distance; causal,
    window, prefix int32 [n_seq] (positions below it are visible to every
    token, those ahead of it included: a prefix-LM mask; the first rows that a
    window keeps only for tokens behind them) and doc int32 [n_seq][positions]
    (other documents are masked). scale 0: 1 / sqrt(hd)."""
    scale: float = 0.0
    softcap: float = 0.0
    slopes: torch.Tensor | None = None
    causal: bool = True
    window: int = 0
    prefix: torch.Tensor | None = None
    doc: torch.Tensor | None = None

    def _at(self, n_seq: int, H: int, dev: int) -> int:
        """The address of the C struct, after the tensors were found to be those of n_seq sequences and H heads on device dev. It is built
        once and lives as long as the score (another thread's call may be reading it): no field depends on the call."""
        made = self.__dict__.get("_made")
        if made is None:
            c = _Score(self.scale, self.softcap, _f32(self.slopes, "slopes"), _i32(self.prefix, "prefix"), _i32(self.doc, "doc"),
                       self.doc.shape[-1] if self.doc is not None else 0, 1 if self.causal else 0, self.window)
            made = self.__dict__.setdefault("_made", (c, C.addressof(c), set()))
        if (n_seq, H, dev) not in made[2]:
            _f32(self.slopes, "slopes", (H,), dev)
            _i32(self.prefix, "prefix", (n_seq,), dev)
            _i32(self.doc, "doc", None, dev)
            if self.doc is not None and (self.doc.dim() != 2 or self.doc.shape[0] != n_seq):
                raise TlmError(-3, f"doc has shape {tuple(self.doc.shape)}, not [{n_seq}][positions]")
            made[2].add((n_seq, H, dev))
        return made[1]


_PLAIN = Score()


class Kv8Cache:
    """K and V pools of one layer (n_pages pages of page_size rows, KV heads
    of hd) in format INT8 or E4M3, one scale per `block` rows; positions=True
    adds the position pool that evicted sequences need."""

    def __init__(self, n_pages: int, KV: int, page_size: int, hd: int, fmt: int = INT8, block: int = 16,
                 positions: bool = False, device="cuda"):
        if fmt not in (INT8, E4M3):
            raise TlmError(-3, f"format {fmt} (int8 1 or e4m3 2)")
        if block <= 0 or page_size % block:
            raise TlmError(-3, f"block {block} does not divide the page of {page_size} rows")
        dt = torch.int8 if fmt == INT8 else torch.float8_e4m3fn
        shape = (n_pages, KV, page_size, hd)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dt) for _ in range(2))
        ks, vs = (torch.zeros((n_pages, KV, page_size // block), device=device) for _ in range(2))
        pos = torch.zeros((n_pages, KV, page_size), dtype=torch.int32, device=device) if positions else None
        self._set(k, v, ks, vs, pos)

    @classmethod
    def from_pools(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                   pos: torch.Tensor | None = None) -> "Kv8Cache":
        """A cache on pools that the caller holds (no copy)."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale, pos)
        return self

    def _set(self, k, v, k_scale, v_scale, pos) -> None:
        if k.dtype not in _FMT or v.dtype != k.dtype:
            raise TlmError(-3, f"code pools must both be int8 or float8_e4m3fn, not {k.dtype} and {v.dtype}")
        if k.dim() != 4 or v.shape != k.shape:
            raise TlmError(-3, f"code pools have shapes {tuple(k.shape)} and {tuple(v.shape)}, not [n_pages][KV][page][hd]")
        n_pages, KV, page, hd = k.shape
        if k_scale.dim() != 3 or k_scale.shape[2] == 0 or page % k_scale.shape[2]:
            raise TlmError(-3, f"scale pools have shape {tuple(k_scale.shape)}, not [n_pages][KV][page / block]")
        blocks = k_scale.shape[2]
        self.k, self.v, self.k_scale, self.v_scale, self.pos = k, v, k_scale, v_scale, pos
        self.KV, self.page_size, self.hd, self.block, self.fmt = KV, page, hd, page // blocks, _FMT[k.dtype]
        self._dev = dev = k.get_device()
        self._c = _Cache(_dev(k, "k"), _ptr(v, "v", dev), _f32(k_scale, "k_scale", (n_pages, KV, blocks), dev),
                         _f32(v_scale, "v_scale", (n_pages, KV, blocks), dev), _i32(pos, "pos", (n_pages, KV, page), dev),
                         self.fmt, n_pages, KV, page, self.block, hd)
        self._p = C.addressof(self._c)
        lib = load()
        self._append, self._read, self._attend = lib.tlmg_kv8_append, lib.tlmg_kv8_read, lib.tlmg_kv8_attend
        self._need, self._select, self._compact = lib.tlmg_kv8_attend_work_bytes, lib.tlmg_kv8_select, lib.tlmg_kv8_compact

    def append(self, k: torch.Tensor, v: torch.Tensor, batch: Kv8Batch) -> None:
        """Stores the batch's new rows k, v [n][KV][hd] (float32, float16 or
        bfloat16)."""
        k, sk, kp = _rows(k, "k", self.KV, self.hd, self._dev)
        v, sv, vp = _rows(v, "v", self.KV, self.hd, self._dev)
        if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
            raise TlmError(-3, f"k and v differ: {k.dtype} x {k.shape[0]} rows, {v.dtype} x {v.shape[0]} rows")
        if sk != sv:
            k, v = k.contiguous(), v.contiguous()
            sk, kp, vp = self.KV * self.hd, k.data_ptr(), v.data_ptr()
        check(self._append(self._p, batch._at(k.shape[0], self._dev), _X_DT[k.dtype], kp, vp, sk, _stream(self._dev)))

    def read(self, page_table: torch.Tensor, row0: torch.Tensor, start: torch.Tensor, total: int,
             k: torch.Tensor | None = None, v: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows row0[s] .. of every sequence as float32 (rows start[s] ..
        start[s + 1] - 1 of the results [total][KV][hd])."""
        n_seq, stride = page_table.shape
        shape = (total, self.KV, self.hd)
        k = torch.empty(shape, dtype=torch.float32, device=self.k.device) if k is None else k
        v = torch.empty_like(k) if v is None else v
        dev = self._dev
        check(self._read(self._p, n_seq, _i32(page_table, "page_table", None, dev), stride, _i32(row0, "row0", (n_seq,), dev),
                         _i32(start, "start", (n_seq + 1,), dev), total, _f32(k, "k", shape, dev), _f32(v, "v", shape, dev),
                         _stream(dev)))
        return k, v

    def attend(self, q: torch.Tensor, batch: Kv8Batch, score: Score | None = None, out: torch.Tensor | None = None,
               lse: bool | torch.Tensor = False, weights: torch.Tensor | None = None):
        """Attention of the batch's tokens q [n][H][hd] over their sequences'
        rows -> out (q's dtype), or (out, lse) with lse. weights float32
        [n_seq][KV][rows >= max_kv] accumulates every row's softmax weights
        (what evict goes by); max_q <= 64 then."""
        shape = q.shape
        if len(shape) != 3:
            raise TlmError(-3, f"q has shape {tuple(shape)}, not [n][H][{self.hd}]")
        n, H = shape[0], shape[1]
        q, sq, qp = _rows(q, "q", H, self.hd, self._dev)
        b = batch._at(n, self._dev)
        s = (score or _PLAIN)._at(batch.n_seq, H, self._dev)
        dt = _X_DT[q.dtype]
        if out is None:
            out = torch.empty(shape, dtype=q.dtype, device=q.device)
        elif out.shape != shape or out.dtype != q.dtype:
            raise TlmError(-3, f"out is {out.dtype} {tuple(out.shape)}, q {q.dtype} {tuple(shape)}")
        lse_t = None
        if lse is not False and lse is not None:
            lse_t = torch.empty((n, H), dtype=torch.float32, device=q.device) if lse is True else lse
        if batch.max_q == 0:    # no sequence may have a token: those that do break the bound
            out.fill_(float("nan"))
            if lse_t is not None:
                lse_t.fill_(float("nan"))
        w_stride = 0
        if weights is not None:
            if weights.dim() != 3 or weights.shape[:2] != (batch.n_seq, self.KV):
                raise TlmError(-3, f"weights have shape {tuple(weights.shape)}, not [{batch.n_seq}][{self.KV}][rows]")
            w_stride = weights.shape[2]
        st = _stream(self._dev)
        call = (self._p, b, s, H, dt, qp, sq, _ptr(out, "out", self._dev), _f32(lse_t, "lse", (n, H), self._dev),
                _f32(weights, "weights", None, self._dev), w_stride)
        rc, dev = TLMG_ERANGE, q.device
        if not _capturing():
            w = _scratch.get((self._dev, st)) or _scratch.setdefault((self._dev, st), _Scratch(dev))
            with w.lock:
                rc = self._attend(*call, w.at, w.size, st)
                if rc == TLMG_ERANGE:                  # what is kept is too small, most likely
                    need = self._need(self._p, b, s, H, dt, 0 if weights is None else 1)
                    if w.size < need <= KEEP:
                        w.grow(need, dev)
                        rc = self._attend(*call, w.at, w.size, st)
        if rc == TLMG_ERANGE:
            need = self._need(self._p, b, s, H, dt, 0 if weights is None else 1)
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            rc = self._attend(*call, work.data_ptr(), need, st)
        check(rc)
        return out if lse_t is None else (out, lse_t)

    def evict(self, weights: torch.Tensor, batch: Kv8Batch, dst_table: torch.Tensor, n_keep: int, sink: int = 0,
              recent: int = 0, dst: "Kv8Cache | None" = None, weights_out: torch.Tensor | None = None,
              rows: torch.Tensor | None = None, lens: torch.Tensor | None = None):
        """Cuts every (sequence, head) to n_keep rows: the first `sink`, the
        last `recent` and those of the largest weights. The rows move into
        dst_table's pages (of `dst`, or of this cache: other pages than
        the sequences hold). Returns (rows int32 [n_seq][KV][n_keep], lens
        int32 [n_seq]): the rows kept, ascending and -1 after the last, and
        the new lengths. weights_out float32 [n_seq][KV][n_keep or more]
        (another buffer than weights) takes the kept rows' weights; its entries
        from n_keep on, which later tokens add theirs to, are left to the caller
        to clear."""
        d = dst or self
        n, dev, on = batch.n_seq, self.k.device, self._dev
        if batch._dev != on or d._dev != on:
            raise TlmError(-3, f"the cache is on cuda:{on}, the batch on cuda:{batch._dev}, the destination on cuda:{d._dev}")
        if weights.dim() != 3 or weights.shape[:2] != (n, self.KV):
            raise TlmError(-3, f"weights have shape {tuple(weights.shape)}, not [{n}][{self.KV}][rows]")
        if dst_table.dim() != 2 or dst_table.shape[0] != n:
            raise TlmError(-3, f"dst_table has shape {tuple(dst_table.shape)}, not [{n}][stride]")
        if weights_out is not None and (weights_out.dim() != 3 or weights_out.shape[:2] != (n, self.KV)):
            raise TlmError(-3, f"weights_out has shape {tuple(weights_out.shape)}, not [{n}][{self.KV}][rows]")
        rows = torch.empty((n, self.KV, max(n_keep, 0)), dtype=torch.int32, device=dev) if rows is None else rows
        lens = torch.empty((n,), dtype=torch.int32, device=dev) if lens is None else lens
        st = _stream(on)
        w, r = _f32(weights, "weights", None, on), _i32(rows, "rows", (n, self.KV, n_keep), on)
        to, wo = _i32(dst_table, "dst_table", None, on), _f32(weights_out, "weights_out", None, on)
        b = batch._c
        check(self._select(n, self.KV, b.kv_len, batch.max_kv, w, weights.shape[2], n_keep, sink, recent, r,
                           _i32(lens, "lens", (n,), on), st))
        check(self._compact(self._p, d._p, n, b.page_table, b.table_stride, b.kv_len, to, dst_table.shape[1], r, n_keep, w,
                            weights.shape[2], wo, 0 if weights_out is None else weights_out.shape[2], st))
        return rows, lens


def _main() -> None:
    """`python -m tierlm_b200.kvcache --prompt N --tokens T --keep R`: one layer's
    serving loop on random rows, a tenth of them near what the tokens ask for. A prompt goes in by chunks (append, then
    attention of the chunk), tokens are decoded one by one while the weights
    that every row receives are accumulated, the sequence is cut to R rows by
    those weights, and decoding goes on in the rows that are left. Prints the
    device time of each part (CUDA events, second of two passes) and how far
    the outputs after the cut are from those of the whole cache."""
    import argparse
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--chunk", type=int, default=2048)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--keep", type=int, default=2048)
    ap.add_argument("--fmt", choices=["int8", "e4m3"], default="int8")
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--softcap", type=float, default=0.0)
    a = ap.parse_args()
    dev = torch.device("cuda:0")
    check(load().tlmg_init(0))
    H, KV, hd, N, T = a.heads, a.kv_heads, a.head_dim, a.prompt, a.tokens
    if a.keep < 36 or N <= 0 or T <= 0 or a.chunk <= 0:
        raise SystemExit("kvcache: prompt, tokens and chunk of at least 1, keep of at least 36 rows")
    whole, cut = -(-(N + 2 * T) // a.page), -(-(a.keep + T) // a.page)
    g = torch.Generator(device=dev).manual_seed(0)
    rnd = lambda n, h: torch.randn((n, h, hd), generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    q, k, v = rnd(N + 2 * T, H), rnd(N + 2 * T, KV), rnd(N + 2 * T, KV)
    u = rnd(1, 1).sign() * (8.0 / hd ** 0.5) ** 0.5     # adds 8 to a score where both have it
    q += u
    k += u * (torch.rand((N + 2 * T, 1, 1), generator=g, device=dev) < 0.1)
    cache = Kv8Cache(whole + cut, KV, a.page, hd, fmt=INT8 if a.fmt == "int8" else E4M3, positions=True, device=dev)
    order = torch.randperm(whole + cut, generator=g, device=dev).to(torch.int32)
    table, cut_table = order[None, :whole].contiguous(), order[None, whole:].contiguous()
    score = Score(softcap=a.softcap)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    one = i32(0, 1)

    def feed(i: int, n: int, tab: torch.Tensor, rows: int, **kw):
        """Tokens i .. i + n - 1 into a sequence that then has `rows` rows."""
        at = torch.arange(i, i + n, dtype=torch.int32, device=dev)
        b = Kv8Batch(tab, one if n == 1 else i32(0, n), i32(rows), n, rows, q_pos=at)
        cache.append(k[i:i + n], v[i:i + n], b)
        return cache.attend(q[i:i + n], b, score, **kw), b

    def timed(what: str, fn, show: bool):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        r = fn()
        e1.record()
        torch.cuda.synchronize()
        if show:
            print(f"{what}: {e0.elapsed_time(e1):.3f} ms")
        return r

    for show in (False, True):
        weights = torch.zeros((1, KV, N + 2 * T), device=dev)
        timed(f"prompt of {N} in chunks of {a.chunk}",
              lambda: [feed(i, min(a.chunk, N - i), table, min(i + a.chunk, N)) for i in range(0, N, a.chunk)], show)
        b = timed(f"{T} tokens, weights accumulated",
                  lambda: [feed(i, 1, table, i + 1, weights=weights)[1] for i in range(N, N + T)], show)[-1]
        rows, lens = timed(f"cut of {N + T} rows to {a.keep}",
                           lambda: cache.evict(weights, b, cut_table, a.keep, sink=4, recent=32), show)
        left = int(lens[0])
        short = timed(f"{T} tokens in {left} rows",
                      lambda: [feed(N + T + i, 1, cut_table, left + i + 1)[0] for i in range(T)], show)
        full = timed(f"{T} tokens in {N + T} rows",
                     lambda: [feed(N + T + i, 1, table, N + T + i + 1)[0] for i in range(T)], show)
    s, f = torch.cat(short).float(), torch.cat(full).float()
    print(f"kept {left} of {N + T} rows a head; |out - whole| / |whole| = {float((s - f).norm() / f.norm()):.3f}")


if __name__ == "__main__":
    _main()
