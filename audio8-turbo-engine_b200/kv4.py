"""A key/value cache held in 4 bits: written with RoPE, read back, attended by decode rows and by packed prompts.

A bf16 cache (the reference's, serve/fast_engine.py:105-106) spends 16 bits an element and decode attention reads all
of it every token; here an element is a 4-bit code with one bf16 scale per 32 of them (4.5 bits). The order of calls in
a layer is that of the bf16 path: the qkv GEMM (``a8_gemm`` with its bias epilogue), ``store`` in place of its RoPE
epilogue, then ``attention`` for decode rows or ``prefill_attention`` for packed prompts.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

BF16, I32 = torch.bfloat16, torch.int32


INT = (1 << 31) - 1      # what a number or a row stride may be: ctypes would cut more to 32 bits, without a word


def _need(ok, what):
    if not ok:
        raise L.A8Error(f"kv4: {what}")


class KV4Cache:
    """`layers` caches of `cache_rows` rows x `nkv` heads x `cache_len` positions x `hd` (64 or 128) on `dev`, empty.
    `buf` (uint8) holds them all; `desc` is the A8KV4 of the C ABI. Tensors given to a call live on the cache's device;
    kernels go to that device's current stream."""

    def __init__(self, cache_rows: int, nkv: int, hd: int, cache_len: int, dev=None, layers: int = 1):
        self.layers, self.cache_rows, self.nkv, self.hd = int(layers), int(cache_rows), int(nkv), int(hd)
        self.cache_len = int(cache_len)
        self.desc = L.A8KV4(None, self.layers, self.cache_rows, self.nkv, self.hd, self.cache_len)
        n = L.load().a8_kv4_bytes(C.byref(self.desc))
        _need(n > 0 and max(self.layers, self.cache_rows, self.nkv, self.hd, self.cache_len) <= INT
              and min(self.layers, self.cache_rows, self.nkv, self.hd, self.cache_len) > 0, f"unsupported shape {(layers, cache_rows, nkv, hd, cache_len)} (hd 64 or 128)")
        self.buf = torch.zeros(n, dtype=torch.uint8, device=torch.device("cuda" if dev is None else dev))
        self.dev = self.buf.device
        self.desc.buf = self.buf.data_ptr()
        if self.dev.type == "cuda":
            if self.dev.index is None:
                self.dev = torch.device("cuda", torch.cuda.current_device())
            # (a torch without CUDA has none of these)
            self._current_device, self._current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
            self._capturing = torch._C._cuda_isCurrentStreamCapturing
        self._ref = C.byref(self.desc)
        self._lib = L.load()
        self._ws = {}
        L.counters.add(self)

    def reset_counters(self):
        """Drop the workspaces of `attention` (not what the cache holds): their tickets are zero between calls, and later
        calls join too early where they are not. The package's `clear_error` calls it."""
        self._ws.clear()

    @property
    def nbytes(self) -> int:
        return self.buf.numel()

    # ---- argument checks: on the host, before anything is launched, and kept lean (a decode step's kernel takes a few
    # microseconds, a check a tenth of one; the C entry points check shapes, strides and alignment again)
    def _rows(self, t, rows, width, what):
        """Row stride of bf16 rows [>= rows, >= width]."""
        shape, (ld, one) = t.shape, t.stride() if t.dim() == 2 else (0, 0)
        if one != 1 or t.dtype is not BF16 or t.device != self.dev or shape[0] < rows or shape[1] < width:
            _need(False, f"{what}: bf16 [at least {rows}, at least {width}] on {self.dev}, rows contiguous")
        # (the row stride of a single row means nothing: torch may give it any value)
        return self._stride(ld, what) if rows > 1 else width

    def _stride(self, ld, what):
        if ld > INT:
            _need(False, f"{what}: a row stride of {ld}")
        return ld

    def _heads(self, t, rows, what):
        """Row stride of bf16 [>= rows, nkv, hd] with contiguous heads."""
        _need(t.dtype is BF16 and t.device == self.dev and t.dim() == 3 and t.shape[0] >= rows
              and t.shape[1:] == (self.nkv, self.hd) and t.stride(2) == 1
              and (self.nkv == 1 or t.stride(1) == self.hd),
              f"{what}: bf16 [at least {rows}, {self.nkv}, {self.hd}] on {self.dev}, heads contiguous")
        return self._stride(t.stride(0), what) if rows > 1 else self.nkv * self.hd

    def _ints(self, t, n, what):
        if t.dtype is not I32 or t.device != self.dev or not t.is_contiguous() or t.numel() < n or n > INT:
            _need(False, f"{what}: {n} contiguous int32 on {self.dev}")
        return t.data_ptr()

    @staticmethod
    def _scale(scale):
        if 0.0 < scale < 1.2e-38:
            _need(False, f"scale {scale}: below the least normal fp32 number")
        return scale

    def _call(self, fn, layer, *args):
        """fn(cache, layer, *args, the current stream of the cache's device)."""
        dev = self.dev.index
        if not 0 <= layer < self.layers:
            _need(False, f"layer {layer} of {self.layers}")
        if dev is None:
            _need(False, "the cache is not on a GPU (there is no CPU fallback)")
        if dev == self._current_device():
            rc = fn(self._ref, layer, *args, self._current_stream(dev))
        else:
            with torch.cuda.device(dev):
                rc = fn(self._ref, layer, *args, self._current_stream(dev))
        if rc:
            L.check(rc, fn.__name__)

    # ---- the operators
    def store(self, qkv, pos, slot=None, *, layer: int = 0, nq: int = 0, cos=None, sin=None, ring: int = 0, q=None):
        """Rows [q | k | v] of qkv [rows, (nq + 2 nkv) hd] into positions pos (int32 [rows]; negative: padding) of cache
        rows slot (int32, None: the row index); with cos / sin [npos, hd] q and k are rotated (rotate_half). Returns the
        query heads [rows, nq hd]: `q` if given (it may be qkv), else a new tensor (None with nq = 0); padding rows of it
        are not written."""
        rows, hd = pos.numel(), self.hd
        ld = self._rows(qkv, rows, (nq + 2 * self.nkv) * hd, "qkv")
        ppos = self._ints(pos, rows, "pos")
        pslot = None if slot is None else self._ints(slot, rows, "slot")
        npos = pcos = psin = None
        if cos is not None and sin is not None:
            npos = cos.shape[0]
            if (cos.dtype is not BF16 or sin.dtype is not BF16 or cos.shape != (npos, hd) or sin.shape != (npos, hd)
                    or not cos.is_contiguous() or not sin.is_contiguous() or cos.device != self.dev
                    or sin.device != self.dev or npos == 0):
                _need(False, f"cos, sin: two contiguous bf16 [npos, {hd}] tables on {self.dev}, npos at least 1")
            pcos, psin = cos.data_ptr(), sin.data_ptr()
        else:
            _need(cos is None and sin is None, "cos and sin come together")
        if not 0 <= ring <= self.cache_len:
            _need(False, f"ring {ring} of a cache of {self.cache_len}")
        ldq = pq = None
        if nq > 0:
            if q is None:
                ldq = nq * hd
                q = torch.empty(rows, ldq, dtype=BF16, device=self.dev)
            else:
                ldq = self._rows(q, rows, nq * hd, "q")
                if rows == 1:                            # (in place asks for one stride)
                    ldq = ld
            pq = q.data_ptr()
        if rows:
            self._call(self._lib.a8_kv4_store, layer, qkv.data_ptr(), ld, nq, pcos, psin, npos or 0, ppos, pslot, rows,
                       ring, pq, ldq or 0)
        return q if nq > 0 else None

    def load(self, pos, slot=None, *, layer: int = 0, k=None, v=None):
        """(k, v) bf16 [rows, nkv, hd] at positions pos of cache rows slot (None: the row index): code * scale, rounded
        once. Given tensors are written in place; rows with a negative position are left as they are (undefined in new
        tensors)."""
        rows = pos.numel()
        ppos = self._ints(pos, rows, "pos")
        pslot = None if slot is None else self._ints(slot, rows, "slot")
        ldk = ldv = self.nkv * self.hd
        if k is None:
            k = torch.empty(rows, self.nkv, self.hd, dtype=BF16, device=self.dev)
        else:
            ldk = self._heads(k, rows, "k")
        if v is None:
            v = torch.empty(rows, self.nkv, self.hd, dtype=BF16, device=self.dev)
        else:
            ldv = self._heads(v, rows, "v")
        if rows:
            self._call(self._lib.a8_kv4_load, layer, ppos, pslot, rows, k.data_ptr(), ldk, v.data_ptr(), ldv)
        return k, v

    def workspace(self, nq: int, rows: int, max_len: int):
        """A workspace (partials, tickets) for `attention` calls up to these sizes; one call at a time uses it."""
        _need(0 < nq <= INT and 0 < rows <= INT and 0 < max_len <= self.cache_len, f"workspace of {nq, rows, max_len}")
        n, t = C.c_longlong(), C.c_int()
        L.check(L.load().a8_kv4_attention_workspace(self._ref, nq, rows, max_len, C.byref(n), C.byref(t)),
                "a8_kv4_attention_workspace")
        return (torch.empty(max(1, n.value), dtype=torch.float32, device=self.dev),
                torch.zeros(max(1, t.value), dtype=torch.int32, device=self.dev))

    def _workspace(self, nq, rows, max_len):
        # Calls on one stream run one after another and share a workspace; every other stream has its own. A captured
        # call gets one of its own inside the graph's memory (cleared by the graph): replays of two graphs may overlap.
        dev = self.dev.index
        if dev is None:
            _need(False, "the cache is not on a GPU (there is no CPU fallback)")
        if dev != self._current_device():                # (whether a stream captures is asked of the current device)
            with torch.cuda.device(dev):
                return self._workspace(nq, rows, max_len)
        capturing = self._capturing()
        key = self._current_stream(dev)
        have = self._ws.get(key)
        if have is None or nq > have[0] or rows > have[1] or max_len > have[2] or capturing:
            if capturing:
                return self._pointers(self.workspace(nq, rows, max_len))
            if have is not None:
                nq, rows, max_len = max(nq, have[0]), max(rows, have[1]), max(max_len, have[2])
            have = self._ws[key] = (nq, rows, max_len, self._pointers(self.workspace(nq, rows, max_len)))
        return have[3]

    @staticmethod
    def _pointers(ws):
        """A workspace as the C call takes it, and the tensors themselves (to keep)."""
        w, t = ws
        return w.data_ptr(), w.numel(), t.data_ptr(), t.numel(), ws

    def attention(self, q, lens, rowmap=None, *, layer: int = 0, max_len: int = 0, scale: float = 0.0, out=None, ws=None):
        """Decode attention: q bf16 [rows, nq hd], row r over keys [0, min(lens[r], max_len)) of cache row rowmap[r]
        (None: r); an empty row gives zeros. max_len bounds every row's keys (0: cache_len). Returns bf16 [rows, nq hd].
        ws: a `workspace()` of the caller's (None: the stream's own)."""
        nq, ldq, ldo, out = self._queries(q, out)
        rows = q.shape[0]
        max_len = max_len or self.cache_len
        if not 0 < max_len <= self.cache_len:
            _need(False, f"max_len {max_len} of a cache of {self.cache_len}")
        plens = self._ints(lens, rows, "lens")           # (the tensors stay referenced until the launch)
        pmap = None if rowmap is None else self._ints(rowmap, rows, "rowmap")
        if rows:
            if ws is not None:
                _need(ws[0].dtype is torch.float32 and ws[1].dtype is I32 and ws[0].device == ws[1].device == self.dev
                      and ws[0].is_contiguous() and ws[1].is_contiguous(),
                      f"ws: the (float32, int32) tensors of workspace() on {self.dev}")
            pw, nw, pt, nt, held = self._workspace(nq, rows, max_len) if ws is None else self._pointers(ws)
            self._call(self._lib.a8_kv4_attention, layer, q.data_ptr(), ldq, nq, plens, pmap, rows, max_len,
                       self._scale(scale), out.data_ptr(), ldo, pw, nw, pt, nt)
        return out

    def _queries(self, q, out):
        """(nq, row stride of q, of out, out) of q [rows, nq hd]."""
        rows, width = q.shape if q.dim() == 2 else (0, -1)
        if width < 0 or width % self.hd:
            _need(False, f"q: [rows, heads of {self.hd}]")
        ldq = self._rows(q, rows, width, "q")
        if out is None:
            return width // self.hd, ldq, width, torch.empty(rows, width, dtype=BF16, device=self.dev)
        return width // self.hd, ldq, self._rows(out, rows, width, "out"), out

    def prefill_attention(self, q, blocks, *, layer: int = 0, scale: float = 0.0, out=None):
        """Packed causal attention: q bf16 [rows, nq hd], blocks int32 [n, 4] = (q0, n, slot, pos0) on the device (the
        rows of `FastEngine.query_blocks`). Rows that no block covers are left as they are. Returns bf16 [rows, nq hd]."""
        nq, ldq, ldo, out = self._queries(q, out)
        rows = q.shape[0]
        _need(blocks.dim() == 2 and blocks.shape[1] == 4, "blocks: int32 [n, 4]")
        n = blocks.shape[0]
        pblocks = self._ints(blocks, 4 * n, "blocks")
        if rows and n:
            self._call(self._lib.a8_kv4_prefill_attention, layer, q.data_ptr(), ldq, nq, pblocks, n, rows,
                       self._scale(scale), out.data_ptr(), ldo)
        return out
