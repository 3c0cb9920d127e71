"""The paged 8-bit KV cache's operators in plain numpy, 64 bits: block tables
and slot maps, the quantizing store, and attention over stored values."""

from __future__ import annotations

import numpy as np

BLOCK = 16


def rope_tables(rows: int, n_rot: int, base: float = 10000.0):
    th = np.arange(rows)[:, None] * base ** (-2.0 * np.arange(n_rot // 2) / n_rot)
    return np.cos(th).astype(np.float32), np.sin(th).astype(np.float32)


def rotate(x, pos, cos, sin, n_rot: int, neox: bool):
    """x [n][heads][hd] at positions pos, in x's precision."""
    x = x.copy()
    hd = x.shape[-1]
    j = np.arange(n_rot // 2)
    i0, i1 = (j, j + hd // 2) if neox else (2 * j, 2 * j + 1)
    c, s = cos[pos][:, None, :].astype(x.dtype), sin[pos][:, None, :].astype(x.dtype)
    a, b = x[..., i0].copy(), x[..., i1].copy()
    x[..., i0] = a * c - b * s
    x[..., i1] = a * s + b * c
    return x


def plan(past, fresh, page: int, table, stack):
    """(table, cu, len, slot, pos, stack) after a step; stack's top is its end."""
    table, stack = table.copy(), list(stack)
    cu, slot, pos = [0], [], []
    for i, (p, f) in enumerate(zip(past, fresh)):
        for col in range(-(-p // page), -(-(p + f) // page)):
            table[i, col] = stack.pop()
        for q in range(p, p + f):
            slot.append(int(table[i, q // page]) * page + q % page)
            pos.append(q)
        cu.append(cu[-1] + f)
    return table, np.array(cu), np.array(past) + np.array(fresh), np.array(slot, np.int64), np.array(pos), stack


class Cache:
    """One layer's K or V: codes [n_pages][hkv][page][hd], scales f32."""

    def __init__(self, n_pages: int, hkv: int, page: int, hd: int):
        self.codes = np.zeros((n_pages, hkv, page, hd), np.int8)
        self.scale = np.zeros((n_pages, hkv, page // BLOCK), np.float32)
        self.page = page

    def store(self, x, slot) -> None:
        """Rows x [n][hkv][hd] f32 at their slots, f32 arithmetic as the header states it."""
        t = 0
        one = np.float32(1)
        while t < len(slot):
            if slot[t] < 0:
                t += 1
                continue
            n = 1
            while t + n < len(slot) and slot[t + n] >= 0 and slot[t + n] // BLOCK == slot[t] // BLOCK:
                n += 1
            pg, off = int(slot[t]) // self.page, int(slot[t]) % self.page
            sub, lead = off // BLOCK, off % BLOCK
            for h in range(x.shape[1]):
                rows = x[t:t + n, h].astype(np.float32)
                fin = np.isfinite(rows)
                amax = np.abs(rows[fin]).max() if fin.any() else np.float32(0)
                before = self.scale[pg, h, sub] if lead else np.float32(0)
                s = max(before, np.float32(amax) * (one / np.float32(127)) if amax >= 2.0 ** -112 else np.float32(0))
                inv = one / s if s > 0 else np.float32(0)
                blk = self.codes[pg, h, sub * BLOCK:(sub + 1) * BLOCK]
                if s > before and lead:
                    blk[:lead] = np.rint(blk[:lead].astype(np.float32) * (before * inv)).astype(np.int8)
                with np.errstate(invalid="ignore", over="ignore"):
                    q = np.clip(np.nan_to_num(np.rint(rows * inv), nan=0.0, posinf=127, neginf=-127), -127, 127)
                for r in range(n):
                    blk[int(slot[t + r]) % BLOCK] = q[r].astype(np.int8)
                self.scale[pg, h, sub] = s
            t += n

    def load(self, slot):
        """f64 rows [n][hkv][hd]."""
        slot = np.asarray(slot)
        pg, off = slot // self.page, slot % self.page
        return self.codes[pg, :, off].astype(np.float64) * self.scale[pg, :, off // BLOCK].astype(np.float64)[..., None]


def attention(q, k: Cache, v: Cache, table, lens, cu, scale, cap=0.0, slopes=None, window=0, prefix=None, first=None):
    """(out f64 [n][n_head][hd], largest |scale q.k| over visible keys); q already rotated, f64."""
    n, n_head, hd = q.shape
    hkv = k.codes.shape[1]
    out = np.zeros((n, n_head, hd))
    top = 0.0
    for i, total in enumerate(lens):
        m = cu[i + 1] - cu[i]
        if m == 0:
            continue
        j = np.arange(total)
        slot = table[i, j // k.page].astype(np.int64) * k.page + j % k.page
        kk, vv = k.load(slot), v.load(slot)
        for r in range(m):
            p = total - m + r
            see = j <= p
            if prefix is not None:
                see |= j < prefix[i]
            if window:
                see &= j > p - window
            if first is not None:
                see &= j >= first[i]
            if not see.any():
                continue
            for h in range(n_head):
                kh = h // (n_head // hkv)
                z = scale * (kk[see][:, kh] @ q[cu[i] + r, h])
                top = max(top, float(np.abs(z).max()))
                if cap:
                    z = cap * np.tanh(z / cap)
                if slopes is not None:
                    z = z - float(slopes[h]) * np.abs(p - j[see])
                w = np.exp(z - z.max())
                out[cu[i] + r, h] = (w / w.sum()) @ vv[see][:, kh]
    return out, top
