"""Device-side paged KV cache and the attention entry points over the C ABI.

``PagedKV`` owns per-layer K/V page pools in HBM (torch device memory is only
the allocator here) and calls libsfa.so for the append, decode and prefill.
It mirrors the engine's KV ownership (src/model/engine/engine.cpp:1253-1286:
per-layer K and V caches owned for the engine's lifetime) with pages in place
of one tensor per layer.  Page tables, seq_len and kv_lo are device int32
tensors, so a call does no host-to-device copy.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import (SFA_AXES_BLOCKS, SFA_AXES_INTERLEAVED, SFA_KV_F16, SFA_KV_F32, SFA_KV_Q8_0, SFA_ROPE_NEOX,
                   SFA_ROPE_NORMAL, SfaKvDesc, SfaRopeDesc)

__all__ = ["PagedKV", "row_bytes", "rope_desc", "SFA_KV_F32", "SFA_KV_F16", "SFA_KV_Q8_0"]


def row_bytes(kv_type: int, head_dim: int) -> int:
    if kv_type == SFA_KV_F32:
        return head_dim * 4
    if kv_type == SFA_KV_F16:
        return head_dim * 2
    if kv_type == SFA_KV_Q8_0:
        return head_dim // 32 * 34
    raise ValueError(f"unsupported kv type {kv_type}")


def rope_desc(head_dim: int, freq_base: float, n_rot: int | None = None, neox: bool = False,
              sections=None, interleaved: bool = False) -> SfaRopeDesc:
    """The rotation of ``norm_rope_append``: the first n_rot elements of a head
    (all by default) in pairs (x[2i], x[2i+1]), or (x[i], x[i + n_rot/2]) with
    ``neox``; ``sections``: the pairs of each axis of a position, in blocks or
    dealt in turn (``interleaved``)."""
    d = SfaRopeDesc()
    d.n_rot = head_dim if n_rot is None else n_rot
    d.pairing = SFA_ROPE_NEOX if neox else SFA_ROPE_NORMAL
    d.freq_base = freq_base
    sections = [d.n_rot // 2] if sections is None else list(sections)
    if not 1 <= len(sections) <= 4:
        raise ValueError("a position has one to four axes")
    d.n_axis = len(sections)
    d.sections[:len(sections)] = sections
    d.layout = SFA_AXES_INTERLEAVED if interleaved else SFA_AXES_BLOCKS
    _lib.check(_lib.load().sfa_rope_desc_check(ctypes.byref(d), head_dim), "rope descriptor")
    return d


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        return _lib.current_stream()
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


_INT32_MAX = 2 ** 31 - 1  # what is larger would be taken modulo 2^32


def _raw_stream(stream, device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else _stream(stream)


def _empty(shape: tuple, like: torch.Tensor, stream, dtype: torch.dtype | None = None) -> torch.Tensor:
    """An uninitialised tensor on `like`'s device (and of its type) in the
    allocator's order of the stream that uses it: freed while the call still
    runs, it is handed on to that stream alone."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(_stream(stream), like.device)
    with torch.cuda.stream(s):
        return like.new_empty(shape, dtype=dtype)


class PagedKV:
    """Per-layer paged K/V pools: k[layer] is [n_pages, page_bytes] uint8."""

    def __init__(self, n_layer: int, n_head: int, n_head_kv: int, head_dim: int, kv_type: int,
                 page_size: int, n_pages: int, device: str | torch.device = "cuda",
                 n_cold_pages: int = 0):
        self.n_layer, self.n_head, self.n_head_kv = n_layer, n_head, n_head_kv
        self.head_dim, self.kv_type, self.page_size = head_dim, kv_type, page_size
        self.n_pages, self.n_cold_pages = n_pages, n_cold_pages
        self.device = torch.device(device)
        self.page_bytes = row_bytes(kv_type, head_dim) * n_head_kv * page_size
        self.k = torch.zeros((n_layer, n_pages, self.page_bytes), dtype=torch.uint8, device=self.device)
        self.v = torch.zeros_like(self.k)
        self._dev = self.k.device  # with its index
        self._index = self.k.get_device()
        self._scale = self.scale
        if n_cold_pages:
            # host-pinned cold pool, readable by the GPU over the host link
            self.k_cold = torch.zeros((n_layer, n_cold_pages, self.page_bytes), dtype=torch.uint8,
                                      pin_memory=True)
            self.v_cold = torch.zeros_like(self.k_cold, pin_memory=True)
        else:
            self.k_cold = self.v_cold = None
        self._ws = None
        self._ws_need = {}
        self._ws_window = {}
        self._descs = [self._make_desc(layer) for layer in range(n_layer)]
        lib = _lib.load()
        _lib.check(lib.sfa_kv_desc_check(ctypes.byref(self.desc(0))), "kv descriptor")

    def desc(self, layer: int) -> SfaKvDesc:
        """The sfa_kv_desc of one layer (built once; pool pointers are stable)."""
        return self._descs[layer]

    def _make_desc(self, layer: int) -> SfaKvDesc:
        d = SfaKvDesc()
        d.n_head, d.n_head_kv, d.head_dim = self.n_head, self.n_head_kv, self.head_dim
        d.page_size, d.kv_type, d.n_pages = self.page_size, self.kv_type, self.n_pages
        d.k_pages = self.k[layer].data_ptr()
        d.v_pages = self.v[layer].data_ptr()
        d.n_cold_pages = self.n_cold_pages
        if self.n_cold_pages:
            d.k_cold = self.k_cold[layer].data_ptr()
            d.v_cold = self.v_cold[layer].data_ptr()
        return d

    @property
    def scale(self) -> float:
        return 1.0 / math.sqrt(self.head_dim)

    # -- workspace -------------------------------------------------------------
    def workspace(self, B: int, max_seq_len: int) -> torch.Tensor:
        lib = _lib.load()
        need = self._ws_need.get((B, max_seq_len))
        if need is None:
            need = lib.sfa_decode_workspace_bytes(ctypes.byref(self.desc(0)), B, max_seq_len)
            if need == 0:
                raise ValueError("invalid decode shape")
            self._ws_need[(B, max_seq_len)] = need
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            _lib.check(lib.sfa_workspace_init(self._ws.data_ptr(), self._ws.numel(), _stream(None)),
                       "workspace init")
        return self._ws

    # -- entry points ------------------------------------------------------------
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor,
               pos: torch.Tensor, page_table: torch.Tensor, stream=None) -> None:
        """k, v [n_tok, Hkv, hd] f32 on device; seq/pos [n_tok] int32."""
        n_tok = int(seq.numel())
        assert k.is_contiguous() and v.is_contiguous() and k.dtype == torch.float32
        assert k.shape == (n_tok, self.n_head_kv, self.head_dim) and v.shape == k.shape
        lib = _lib.load()
        d = self.desc(layer)
        _lib.check(lib.sfa_kv_append(ctypes.byref(d), k.data_ptr(), v.data_ptr(), seq.data_ptr(),
                                     pos.data_ptr(), n_tok, page_table.data_ptr(),
                                     int(page_table.shape[-1]), _stream(stream)), "sfa_kv_append")

    def rope_append(self, layer: int, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                    seq: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor, freq_base: float,
                    stream=None) -> None:
        """Fused RoPE NORMAL + append: q [n_tok, Hq, hd] (rotated in place, or
        None), k pre-RoPE and v raw [n_tok, Hkv, hd] f32 on device."""
        n_tok = int(seq.numel())
        assert k.is_contiguous() and v.is_contiguous() and k.dtype == torch.float32
        assert k.shape == (n_tok, self.n_head_kv, self.head_dim) and v.shape == k.shape
        if q is not None:
            assert q.is_contiguous() and q.dtype == torch.float32
            assert q.shape == (n_tok, self.n_head, self.head_dim)
        lib = _lib.load()
        d = self.desc(layer)
        _lib.check(lib.sfa_rope_kv_append(ctypes.byref(d), _ptr(q), k.data_ptr(), v.data_ptr(),
                                          seq.data_ptr(), pos.data_ptr(), n_tok, page_table.data_ptr(),
                                          int(page_table.shape[-1]), float(freq_base), _stream(stream)),
                   "sfa_rope_kv_append")

    def qkv_rope_append(self, layer: int, w_qkv: torch.Tensor, x: torch.Tensor, seq: torch.Tensor,
                        pos: torch.Tensor, page_table: torch.Tensor, freq_base: float,
                        q: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """The stacked Q/K/V product of x [n_tok, n_embd] (w_qkv
        [(Hq + 2 Hkv) hd, n_embd], f32 or f16), RoPE and the append in one
        launch -> q [n_tok, Hq, hd] rotated."""
        from .layer import weight_type
        n_tok = int(seq.numel())
        n_embd = int(x.shape[-1])
        assert x.is_contiguous() and x.dtype == torch.float32 and x.shape == (n_tok, n_embd)
        assert w_qkv.is_contiguous() and w_qkv.shape == ((self.n_head + 2 * self.n_head_kv) * self.head_dim, n_embd)
        if q is None:
            q = torch.empty((n_tok, self.n_head, self.head_dim), dtype=torch.float32, device=x.device)
        assert q.is_contiguous() and q.dtype == torch.float32 and q.shape == (n_tok, self.n_head, self.head_dim)
        lib = _lib.load()
        d = self.desc(layer)
        _lib.check(lib.sfa_qkv_rope_kv_append(ctypes.byref(d), w_qkv.data_ptr(), weight_type(w_qkv), x.data_ptr(),
                                              n_embd, q.data_ptr(), seq.data_ptr(), pos.data_ptr(), n_tok,
                                              page_table.data_ptr(), int(page_table.shape[-1]), float(freq_base),
                                              _stream(stream)),
                   "sfa_qkv_rope_kv_append")
        return q

    def decode(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, seq_len: torch.Tensor,
               max_seq_len: int, kv_lo: torch.Tensor | None = None, out: torch.Tensor | None = None,
               scale: float | None = None, stream=None, split_end_event=None) -> torch.Tensor:
        """q [B, Hq, hd] f32 -> out [B, Hq*hd] f32.  With `split_end_event` the
        two passes are issued separately and the event is recorded between
        them (timing of the split-K pass)."""
        B = int(seq_len.numel())
        assert q.is_contiguous() and q.dtype == torch.float32
        assert q.shape == (B, self.n_head, self.head_dim)
        assert page_table.dtype == torch.int32 and page_table.shape[0] == B
        if out is None:
            out = torch.empty((B, self.n_head * self.head_dim), dtype=torch.float32, device=q.device)
        ws = self.workspace(B, max_seq_len)
        lib = _lib.load()
        d = self._descs[layer]
        args = (ctypes.byref(d), q.data_ptr(), out.data_ptr(), page_table.data_ptr(),
                int(page_table.shape[1]), seq_len.data_ptr(), _ptr(kv_lo), B, int(max_seq_len),
                float(scale if scale is not None else self.scale), ws.data_ptr(), ws.numel(),
                _stream(stream))
        if split_end_event is None:
            _lib.check(lib.sfa_attn_decode(*args), "sfa_attn_decode")
        else:
            _lib.check(lib.sfa_attn_decode_split(*args), "sfa_attn_decode_split")
            split_end_event.record()
            _lib.check(lib.sfa_attn_decode_merge(*args), "sfa_attn_decode_merge")
        return out

    def decode_append(self, layer: int, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor,
                      page_table: torch.Tensor, seq_len: torch.Tensor, max_seq_len: int,
                      kv_lo: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      scale: float | None = None, stream=None) -> torch.Tensor:
        """Appends each sequence's new token (k, v [B, Hkv, hd] f32, token b at
        position seq_len[b] - 1) and attends: out [B, Hq*hd] f32.  F16 or F32 pools."""
        B = int(seq_len.numel())
        assert q.is_contiguous() and q.dtype == torch.float32 and q.shape == (B, self.n_head, self.head_dim)
        for t in (k, v):
            assert t.is_contiguous() and t.dtype == torch.float32 and t.shape == (B, self.n_head_kv, self.head_dim)
        assert page_table.dtype == torch.int32 and page_table.shape[0] == B
        if out is None:
            out = torch.empty((B, self.n_head * self.head_dim), dtype=torch.float32, device=q.device)
        ws = self.workspace(B, max_seq_len)
        lib = _lib.load()
        _lib.check(lib.sfa_attn_decode_append(ctypes.byref(self._descs[layer]), k.data_ptr(), v.data_ptr(),
                                              q.data_ptr(), out.data_ptr(), page_table.data_ptr(),
                                              int(page_table.shape[1]), seq_len.data_ptr(), _ptr(kv_lo), B,
                                              int(max_seq_len),
                                              float(scale if scale is not None else self.scale),
                                              ws.data_ptr(), ws.numel(), _stream(stream)),
                   "sfa_attn_decode_append")
        return out

    def prefill(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, q_pos0: int,
                kv_lo: int = 0, out: torch.Tensor | None = None, scale: float | None = None,
                stream=None) -> torch.Tensor:
        """q [T, Hq, hd] f32 of one sequence -> out [T, Hq*hd] f32."""
        T = int(q.shape[0])
        assert q.is_contiguous() and q.dtype == torch.float32
        if out is None:
            out = torch.empty((T, self.n_head * self.head_dim), dtype=torch.float32, device=q.device)
        lib = _lib.load()
        d = self.desc(layer)
        _lib.check(lib.sfa_attn_prefill(ctypes.byref(d), q.data_ptr(), out.data_ptr(),
                                        page_table.data_ptr(), int(page_table.numel()),
                                        int(q_pos0), T, int(kv_lo),
                                        float(scale if scale is not None else self.scale),
                                        _stream(stream)), "sfa_attn_prefill")
        return out

    # -- windowed models: head norms and rotations on the append, window + sinks ----
    # (the checks are spelled out: where a launch takes 4 us, a helper call per
    # tensor would take as much again)
    def _bad(self, what: str, dtype: str, shape: str) -> ValueError:
        return ValueError(f"{what} must be a contiguous {dtype} tensor {shape} on {self._dev}")

    def _heads(self, t: torch.Tensor, what: str, n_tok: int, heads: int) -> int:
        """Checks [n_tok, heads, hd] f32 rows, whole within a token; the stride between tokens."""
        if t.dtype is not torch.float32 or t.get_device() != self._index or t.shape != (n_tok, heads, self.head_dim):
            raise ValueError(f"{what} must be float32 [{n_tok}, {heads}, {self.head_dim}] on {self._dev}")
        step, head, one = t.stride()
        if one != 1 or (heads > 1 and head != self.head_dim):
            raise ValueError(f"{what}: the heads of a token must lie one after the other")
        return step

    def norm_rope_append(self, layer: int, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                         seq: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor, rope: SfaRopeDesc,
                         q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                         eps: float = 1e-6, rope_pos: torch.Tensor | None = None,
                         q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor | None:
        """Norms the heads of Q and K (q_norm, k_norm [hd], each optional),
        rotates them by ``rope`` and appends K and V; returns the rotated Q
        [n_tok, Hq, hd] (``q_out``, which may be a contiguous q itself).
        q [n_tok, Hq, hd] (or None), k, v [n_tok, Hkv, hd] f32 may be slices of
        the stacked Q/K/V rows; rope_pos [n_axis, n_tok] int32 (default: pos on
        every axis)."""
        i32, dev, hd = torch.int32, self._index, self.head_dim
        if torch.cuda.current_device() != dev:
            with torch.cuda.device(dev):
                return self.norm_rope_append(layer, q, k, v, seq, pos, page_table, rope, q_norm, k_norm, eps, rope_pos,
                                             q_out, stream)
        n_tok = seq.numel()
        ks = self._heads(k, "k", n_tok, self.n_head_kv)
        vs = self._heads(v, "v", n_tok, self.n_head_kv)
        if seq.dtype is not i32 or seq.get_device() != dev or not seq.is_contiguous():
            raise self._bad("seq", "int32", "[n_tok]")
        if pos.dtype is not i32 or pos.get_device() != dev or not pos.is_contiguous() or pos.numel() != n_tok:
            raise self._bad("pos", "int32", f"[{n_tok}]")
        if page_table.dtype is not i32 or page_table.get_device() != dev or not page_table.is_contiguous():
            raise self._bad("page_table", "int32", "[n_seq, max_pages]")
        qs, qp, op = 0, None, None
        if q is not None:
            qs, qp = self._heads(q, "q", n_tok, self.n_head), q.data_ptr()
            if q_out is None:
                q_out = _empty((n_tok, self.n_head, hd), q, stream)
            elif self._heads(q_out, "q_out", n_tok, self.n_head) != self.n_head * hd and n_tok > 1:
                raise self._bad("q_out", "float32", f"[{n_tok}, {self.n_head}, {hd}]")
            op = q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        wq = wk = rp = None
        if q_norm is not None:
            if q_norm.dtype is not torch.float32 or q_norm.get_device() != dev or q_norm.shape != (hd,) or not q_norm.is_contiguous():
                raise self._bad("q_norm", "float32", f"[{hd}]")
            wq = q_norm.data_ptr()
        if k_norm is not None:
            if k_norm.dtype is not torch.float32 or k_norm.get_device() != dev or k_norm.shape != (hd,) or not k_norm.is_contiguous():
                raise self._bad("k_norm", "float32", f"[{hd}]")
            wk = k_norm.data_ptr()
        if rope_pos is not None:
            if (rope_pos.dtype is not i32 or rope_pos.get_device() != dev or not rope_pos.is_contiguous()
                    or rope_pos.shape != (rope.n_axis, n_tok)):
                raise self._bad("rope_pos", "int32", f"[{rope.n_axis}, {n_tok}]")
            rp = rope_pos.data_ptr()
        rc = _lib.load().sfa_norm_rope_kv_append(
            self._descs[layer], rope, qp, qs, op, k.data_ptr(), ks, v.data_ptr(), vs, wq, wk, eps, seq.data_ptr(),
            pos.data_ptr(), rp, n_tok, page_table.data_ptr(), page_table.shape[-1], _raw_stream(stream, dev))
        if rc:
            _lib.check(rc, "sfa_norm_rope_kv_append")
        return q_out

    def _rows(self, q: torch.Tensor, out: torch.Tensor | None, n: int, stream) -> torch.Tensor:
        """Checks q [n, Hq, hd] and out [n, Hq*hd]; out, a new one by default."""
        Hq, hd = self.n_head, self.head_dim
        if q.dtype is not torch.float32 or q.get_device() != self._index or q.shape != (n, Hq, hd) or not q.is_contiguous():
            raise self._bad("q", "float32", f"[{n}, {Hq}, {hd}]")
        if out is None:
            return _empty((n, Hq * hd), q, stream)
        if out.dtype is not torch.float32 or out.get_device() != self._index or out.shape != (n, Hq * hd) or not out.is_contiguous():
            raise self._bad("out", "float32", f"[{n}, {Hq * hd}]")
        return out

    def decode_window(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, seq_len: torch.Tensor,
                      max_seq_len: int, window: int, n_sink: int = 0, out: torch.Tensor | None = None,
                      scale: float | None = None, stream=None) -> torch.Tensor:
        """q [B, Hq, hd] f32 -> out [B, Hq*hd] f32: the token at seq_len[b] - 1
        attends the last ``window`` positions and the first ``n_sink``.  The
        workspace is the call's own."""
        i32, dev = torch.int32, self._index
        if torch.cuda.current_device() != dev:
            with torch.cuda.device(dev):
                return self.decode_window(layer, q, page_table, seq_len, max_seq_len, window, n_sink, out, scale, stream)
        B = seq_len.numel()
        out = self._rows(q, out, B, stream)
        if seq_len.dtype is not i32 or seq_len.get_device() != dev or not seq_len.is_contiguous():
            raise self._bad("seq_len", "int32", "[B]")
        if (page_table.dtype is not i32 or page_table.get_device() != dev or page_table.dim() != 2
                or page_table.shape[0] != B or not page_table.is_contiguous()):
            raise self._bad("page_table", "int32", f"[{B}, max_pages]")
        if max(max_seq_len, window, n_sink) > _INT32_MAX:
            raise ValueError("max_seq_len, window and n_sink are 32-bit")
        lib, d = _lib.load(), self._descs[layer]
        key = (B, max_seq_len, window, n_sink)
        need = self._ws_window.get(key)
        if need is None:
            if len(self._ws_window) >= 1024:
                self._ws_window.clear()
            need = self._ws_window[key] = lib.sfa_decode_window_workspace_bytes(d, *key)
        ws = _empty((need,), out, stream, torch.uint8)
        rc = lib.sfa_attn_decode_window(
            d, q.data_ptr(), out.data_ptr(), page_table.data_ptr(), page_table.shape[1], seq_len.data_ptr(), window,
            n_sink, B, max_seq_len, self._scale if scale is None else scale, ws.data_ptr(), need, _raw_stream(stream, dev))
        if rc:
            _lib.check(rc, "sfa_attn_decode_window")
        return out

    def prefill_window(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, q_pos0: int, window: int,
                       n_sink: int = 0, out: torch.Tensor | None = None, scale: float | None = None,
                       stream=None) -> torch.Tensor:
        """q [T, Hq, hd] f32 of one sequence -> out [T, Hq*hd] f32: the token at
        position t attends the ``window`` positions up to t and the first
        ``n_sink``.  The workspace is the call's own."""
        dev = self._index
        if torch.cuda.current_device() != dev:
            with torch.cuda.device(dev):
                return self.prefill_window(layer, q, page_table, q_pos0, window, n_sink, out, scale, stream)
        T = q.shape[0]
        out = self._rows(q, out, T, stream)
        if page_table.dtype is not torch.int32 or page_table.get_device() != dev or page_table.dim() != 1 or not page_table.is_contiguous():
            raise self._bad("page_table", "int32", "[max_pages]")
        if max(q_pos0, window, n_sink) > _INT32_MAX:
            raise ValueError("q_pos0, window and n_sink are 32-bit")
        lib, d = _lib.load(), self._descs[layer]
        need = lib.sfa_prefill_window_workspace_bytes(d, q_pos0, T, window, n_sink)
        ws = _empty((need,), out, stream, torch.uint8) if need else None
        rc = lib.sfa_attn_prefill_window(
            d, q.data_ptr(), out.data_ptr(), page_table.data_ptr(), page_table.shape[0], q_pos0, T, window, n_sink,
            self._scale if scale is None else scale, _ptr(ws), need, _raw_stream(stream, dev))
        if rc:
            _lib.check(rc, "sfa_attn_prefill_window")
        return out
