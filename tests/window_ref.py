"""64-bit references of the windowed attention node: head norms, rotations and
the append by their formulas, attention by a mask over every position."""
from __future__ import annotations

import math

import numpy as np
import torch

from strataflow_amd.paged_kv import SFA_KV_F16, SFA_KV_F32, SFA_KV_Q8_0, PagedKV, row_bytes

EPS24 = 2.0 ** -24  # half a step of f32, relative


def axes_of(n_pairs, sections, interleaved):
    """Axis of each pair, dealt one pair at a time."""
    if not sections:
        return [0] * n_pairs
    left, out = list(sections), []
    for i in range(n_pairs):
        if interleaved:
            a = i % len(sections)
            a = a if a == 0 or left[a] > 0 else 0
        else:
            a = next(j for j in range(len(left)) if left[j] > 0)
        left[a] -= 1
        out.append(a)
    return out


def norm_rope(x, weight, eps, pos, n_rot, base, neox, sections=None, interleaved=False):
    """x [n, heads, hd] f64 -> normed and rotated; pos [n_axis, n]."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    half = n_rot // 2
    ax = axes_of(half, sections, interleaved)
    y = x.copy()
    for i in range(half):
        ang = pos[ax[i]].astype(np.float64) * float(base) ** (-2.0 * i / n_rot)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def decode_rows(raw, kv_type, hd):
    """Row bytes [..., row_bytes] -> f64 values [..., hd]."""
    raw = np.ascontiguousarray(raw)
    if kv_type == SFA_KV_F32:
        return raw.view(np.float32).astype(np.float64)
    if kv_type == SFA_KV_F16:
        return raw.view(np.float16).astype(np.float64)
    blk = raw.reshape(*raw.shape[:-1], hd // 32, 34)
    d = np.ascontiguousarray(blk[..., :2]).view(np.float16).astype(np.float64)
    q = np.ascontiguousarray(blk[..., 2:]).view(np.int8).astype(np.float64)
    return (d * q).reshape(*raw.shape[:-1], hd)


def encode_rows(x, kv_type):
    """f32 values [..., hd] -> row bytes (any row a cache may hold; the append's own rounding is tested apart)."""
    x = np.ascontiguousarray(x, np.float32)
    if kv_type == SFA_KV_F32:
        return x.view(np.uint8)
    if kv_type == SFA_KV_F16:
        return x.astype(np.float16).view(np.uint8)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    d = np.abs(b).max(-1, keepdims=True) / 127
    q = np.rint(b / np.where(d > 0, d, 1)).astype(np.int8)
    blk = np.concatenate([d.astype(np.float16).view(np.uint8), q.view(np.uint8)], -1)
    return blk.reshape(*x.shape[:-1], x.shape[-1] // 32 * 34)


class Cache:
    """A paged cache of random rows on the host and the device.  Rows that no call may see are bytes
    that read as NaN; `there` [B, n] bool says which positions hold values."""

    def __init__(self, *, lens, there=None, n_head=8, n_head_kv=2, head_dim=64, page_size=64, kv_type=SFA_KV_F16, seed=0,
                 cold=0, boost=None, max_pages=None, drop=()):
        rng = np.random.default_rng(seed)
        self.Hq, self.Hkv, self.hd, self.ps, self.kv_type = n_head, n_head_kv, head_dim, page_size, kv_type
        self.lens = list(lens)
        B = len(self.lens)
        rb = row_bytes(kv_type, head_dim)
        need = [max(0, -(-n // page_size)) for n in self.lens]
        mp = max_pages or max(max(need), 1)
        total = sum(need)
        n_cold = min(cold, total)
        n_dev = total - n_cold + 3
        ids = [int(i) for i in rng.permutation(n_dev)[:total - n_cold]] + [-2 - i for i in range(n_cold)]
        ids = [ids[i] for i in rng.permutation(total)]
        self.table = np.full((B, mp), -1, np.int32)
        self.kv = PagedKV(1, n_head, n_head_kv, head_dim, kv_type, page_size, n_dev, n_cold_pages=n_cold)
        shape = (n_dev, page_size, n_head_kv, rb)
        dev = [np.full(shape, 0xFF, np.uint8) for _ in range(2)]  # 0xFFFF.. reads as NaN (Q8_0: a NaN scale)
        cold_np = [np.full((n_cold,) + shape[1:], 0xFF, np.uint8) for _ in range(2)]
        self.k = [None] * B
        self.v = [None] * B
        for b, n in enumerate(self.lens):
            x = [rng.standard_normal((n, n_head_kv, head_dim)).astype(np.float32) for _ in range(2)]
            if boost is not None and n:
                x[0][:: boost[0]] *= boost[1]
            rows = [encode_rows(y, kv_type) for y in x]
            self.k[b], self.v[b] = (decode_rows(r, kv_type, head_dim) for r in rows)
            ok = np.ones(n, bool) if there is None else there(b, np.arange(n))
            for lp in range(need[b]):
                i = ids.pop()
                if (b, lp) in drop:
                    continue
                sl = slice(lp * page_size, min(n, (lp + 1) * page_size))
                if not ok[sl].any():
                    continue  # a page that no call needs is not there
                self.table[b, lp] = i
                for w in range(2):
                    page = dev[w][i] if i >= 0 else cold_np[w][-2 - i]
                    at = np.nonzero(ok[sl])[0]
                    page[at] = rows[w][sl][at]
        # a page that was dropped is not attended
        self.gone = [np.repeat(self.table[b] == -1, page_size) for b in range(B)]
        for w, t in ((0, self.kv.k), (1, self.kv.v)):
            t[0].copy_(torch.from_numpy(dev[w].reshape(n_dev, -1)))
        if n_cold:
            self.kv.k_cold[0].copy_(torch.from_numpy(cold_np[0].reshape(n_cold, -1)))
            self.kv.v_cold[0].copy_(torch.from_numpy(cold_np[1].reshape(n_cold, -1)))
        self.t_table = torch.from_numpy(self.table).cuda()
        self.rng = rng

    def queries(self, n):
        return self.rng.standard_normal((n, self.Hq, self.hd)).astype(np.float32)

    def attend(self, b, q, tokens, window, n_sink, scale=None):
        """f64 attention of q [n, Hq, hd] at positions `tokens` of sequence b: [n, Hq*hd], and a bound on
        what 32-bit arithmetic may be off by, per token and head."""
        scale = 1.0 / math.sqrt(self.hd) if scale is None else scale
        g = self.Hq // self.Hkv
        tokens = np.asarray(tokens)
        n_pos = min(len(self.k[b]), self.table.shape[1] * self.ps)
        p = np.arange(n_pos)
        sees = (p[None] <= tokens[:, None]) & ((p[None] < n_sink) | (p[None] > tokens[:, None].astype(np.int64) - window))
        sees &= ~self.gone[b][None, :n_pos]
        out = np.zeros((len(tokens), self.Hq, self.hd))
        bound = np.zeros((len(tokens), self.Hq, 1))
        for h in range(self.Hq):
            k, v = self.k[b][:n_pos, h // g], self.v[b][:n_pos, h // g]
            s = np.where(sees, (q[:, h].astype(np.float64) @ k.T) * scale, -np.inf)
            m = s.max(1, keepdims=True, initial=-np.inf)
            e = np.exp(s - np.where(np.isinf(m), 0, m))
            z = e.sum(1, keepdims=True)
            w = e / np.where(z == 0, 1, z)
            out[:, h] = w @ np.where(sees.any(0)[:, None], v, 0)
            # a score's 32-bit error is at most (hd + 4) half steps of its terms' sum; a weight is off by twice
            # the largest of them, its own exp, the two sums over n positions and the products by a few more
            terms = np.abs(q[:, h].astype(np.float64)) @ np.abs(k.T) * scale
            worst = np.where(sees, terms, 0).max(1, initial=0)
            seen = np.where(sees.any(0)[:, None], np.abs(v), 0).max(initial=0)
            bound[:, h, 0] = (2 * (self.hd + 4) * worst + 2 * np.sqrt(sees.sum(1)) + 16) * EPS24 * seen
        return out.reshape(len(tokens), -1), np.broadcast_to(bound, out.shape).reshape(len(tokens), -1)


def check(got, want, bound, hd):
    """Every value within its bound, and the whole within what independent roundings give: a score's error
    is some sqrt(hd) half steps of a typical sum of terms (at most eight here)."""
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert (off <= bound + 1e-30).all(), f"largest excess {np.max(off - bound)}"
    rel = np.linalg.norm(off) / max(np.linalg.norm(want), 1e-30)
    assert rel <= 8 * math.sqrt(hd) * EPS24, rel
