"""The 4-bit paged KV cache by its definition, in numpy and 64 bits: the oracle of the
b2_kv4_* operators (include/b2q4nx.h gives their contracts).

A pool is uint8 [n_pages][n_kv_heads][page / 16][D / 64][1152]; `unpack` and `pack` know the
order of a cell's bytes, everything else works on codes and (d, m) pairs."""

from __future__ import annotations

import numpy as np
from ml_dtypes import bfloat16

CELL, TILE, GROUP = 1152, 16, 64
D_MIN = 2.0 ** -40


def _places() -> tuple[np.ndarray, np.ndarray]:
    """Byte [2][16][64] of each (K or V, token, dim)'s code in a cell (low nibble for even
    dims), and of each (d, m) pair [2][16]."""
    t, d = np.meshgrid(np.arange(16), np.arange(64), indexing="ij")
    k = t % 8 * 64 + d // 16 * 16 + t // 8 * 8 + d % 16 // 2
    v = 512 + d // 8 * 64 + t % 8 // 2 * 16 + t // 8 * 8 + d // 4 % 2 * 4 + t % 2 * 2 + d % 4 // 2
    m = np.arange(16) % 8 * 8 + np.arange(16) // 8 * 4
    return np.stack([k, v]), np.stack([1024 + m, 1088 + m])


CODE_AT, META_AT = _places()


def bf16(x) -> np.ndarray:
    """Rounded to bf16 (through fp32, as a cast from 64 bits goes), as fp64."""
    with np.errstate(invalid="ignore", over="ignore"):
        return np.asarray(x, np.float64).astype(np.float32).astype(bfloat16).astype(np.float64)


def unpack(cells: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Cells [..., 1152] -> codes [..., 2, 16, 64] and (d, m) [..., 2, 16, 2]."""
    code = cells[..., CODE_AT] >> (4 * (np.arange(64) % 2)).astype(np.uint8) & 15
    at = META_AT[..., None] + np.arange(4)
    meta = np.ascontiguousarray(cells[..., at]).view(bfloat16).astype(np.float64)
    return code, meta


def pack(code: np.ndarray, meta: np.ndarray) -> np.ndarray:
    """The inverse of unpack."""
    cells = np.zeros((*code.shape[:-3], CELL), np.uint8)
    cells[..., CODE_AT[..., 0::2]] = code[..., 0::2] | code[..., 1::2] << 4
    at = META_AT[..., None] + np.arange(4)
    cells[..., at] = np.ascontiguousarray(meta.astype(bfloat16)).view(np.uint8)
    return cells


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """x fp64 [..., 64] -> codes [..., 64], (d, m) [..., 2]; a group with a value that is not
    finite is NaN throughout."""
    bad = ~np.isfinite(x.astype(np.float32)).all(-1)
    y = np.where(bad[..., None], 0.0, x)
    m = bf16(y.min(-1))
    d = np.maximum(bf16((y.max(-1) - m) / 15), D_MIN)
    code = np.zeros(x.shape, np.uint8)
    for j in range(15):  # one up at each border between two codes: j + 1/2 steps
        code += (y - m[..., None] >= (j + 0.5) * d[..., None]).astype(np.uint8)
    code[bad] = 0
    return code, np.stack([np.where(bad, D_MIN, d), np.where(bad, np.nan, m)], -1)


def rotate(x: np.ndarray, pos: int, theta: float | None) -> np.ndarray:
    """Half-split rotation of [..., D] at a position, in fp64."""
    x = np.asarray(x, np.float64)
    if theta is None:
        return x
    half = x.shape[-1] // 2
    a = pos * float(theta) ** (-2.0 * np.arange(half) / (2 * half))
    c, s = np.cos(a), np.sin(a)
    return np.concatenate([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)


class Cache:
    """A pool with its summaries, in host memory."""

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, page: int):
        self.hkv, self.dim, self.page = n_kv_heads, head_dim, page
        shape = (n_pages, n_kv_heads, page // TILE, head_dim // GROUP)
        self.code = np.zeros((*shape, 2, TILE, GROUP), np.uint8)
        self.meta = np.zeros((*shape, 2, TILE, 2), np.float64)
        self.summary = np.zeros((n_pages, n_kv_heads, 2, head_dim), np.float64)

    @classmethod
    def of(cls, pool: np.ndarray, head_dim: int, summary: np.ndarray | None = None) -> "Cache":
        n, hkv, nbytes = pool.shape
        c = cls(n, hkv, head_dim, nbytes // CELL // (head_dim // GROUP) * TILE)
        c.code, c.meta = unpack(pool.reshape(*c.code.shape[:4], CELL))
        if summary is not None:
            c.summary = np.asarray(summary, np.float64).copy()
        return c

    def pool(self) -> np.ndarray:
        return pack(self.code, self.meta).reshape(*self.code.shape[:2], -1)

    def values(self, which: int, pages) -> np.ndarray:
        """K (0) or V (1) of pages, [Hkv, len(pages) * page, D]."""
        v = self.code[pages, :, :, :, which].astype(np.float64) * self.meta[pages, :, :, :, which, :, :1] \
            + self.meta[pages, :, :, :, which, :, 1:]
        v = v.transpose(1, 0, 2, 4, 3, 5)  # [hkv, page, tile, token, group, 64]
        return v.reshape(self.hkv, len(pages) * self.page, self.dim)

    def append(self, k, v, table, pos, cu=None, theta=None) -> None:
        rows = len(k)
        cu = np.arange(rows + 1) if cu is None else cu
        for b in range(len(pos)):
            fresh = {}
            for r in range(cu[b], cu[b + 1]):
                if pos[b] < 0:
                    continue
                p = int(pos[b]) + r - cu[b]
                at, off = table[b, p // self.page], p % self.page
                key = rotate(np.asarray(k[r], np.float64).reshape(self.hkv, self.dim), p, theta)
                for which, x in ((0, key), (1, np.asarray(v[r], np.float64).reshape(self.hkv, self.dim))):
                    code, meta = quantise(x.reshape(self.hkv, -1, GROUP))
                    self.code[at, :, off // TILE, :, which, off % TILE] = code
                    self.meta[at, :, off // TILE, :, which, off % TILE] = meta
                fresh.setdefault((at, p // self.page), []).append((off, bf16(key)))
            for (at, _), got in fresh.items():
                keys = np.stack([x for _, x in got])
                low, high = np.fmin.reduce(keys), np.fmax.reduce(keys)
                if got[0][0] > 0:
                    low, high = np.fmin(low, self.summary[at, :, 0]), np.fmax(high, self.summary[at, :, 1])
                self.summary[at] = np.stack([low, high], 1)

    def gather(self, table_row, start: int, n: int) -> tuple[np.ndarray, np.ndarray]:
        """Tokens start .. start + n - 1 as [n, Hkv * D]."""
        pages = table_row[start // self.page:(start + n - 1) // self.page + 1]
        off = start % self.page
        return tuple(self.values(w, pages)[:, off:off + n].transpose(1, 0, 2).reshape(n, -1) for w in (0, 1))

    def decode(self, q, table, pos, theta=None, scale=None, sel=None) -> np.ndarray:
        """[B, Hq, D] fp64; q [B, Hq, D]."""
        q = np.asarray(q, np.float64)
        bsz, hq, dim = q.shape
        grp, out = hq // self.hkv, np.zeros(q.shape)
        scale = dim ** -0.5 if scale is None else scale
        for b in range(bsz):
            n = int(pos[b]) + 1
            if n < 1:
                continue
            turned = rotate(q[b], n - 1, theta)
            pages = table[b, :(n - 1) // self.page + 1]
            k, v = self.values(0, pages), self.values(1, pages)
            token = np.arange(k.shape[1])
            for h in range(self.hkv):
                seen = token < n
                if sel is not None:
                    seen &= np.isin(token // self.page, [p for p in sel[b, h] if p >= 0])
                if not seen.any():
                    continue
                for j in range(grp):
                    s = k[h, seen] @ turned[h * grp + j] * scale
                    w = np.exp(s - s.max())
                    out[b, h * grp + j] = w @ v[h, seen] / w.sum()
        return out

    def select(self, q, table, pos, n_sel: int, theta=None) -> np.ndarray:
        """[B, Hkv, n_sel] page indices."""
        q = np.asarray(q, np.float64)
        bsz, hq, _ = q.shape
        grp, out = hq // self.hkv, np.full((bsz, self.hkv, n_sel), -1, np.int32)
        for b in range(bsz):
            if pos[b] < 0:
                continue
            last = int(pos[b]) // self.page
            turned = rotate(q[b], int(pos[b]), theta)
            for h in range(self.hkv):
                near = self.summary[table[b, :last + 1], h]
                bound = np.max([np.maximum(x * near[:, 0], x * near[:, 1]).sum(-1)
                                for x in turned[h * grp:(h + 1) * grp]], 0)
                order = sorted(range(last + 1), key=lambda p: (p != last, -bound[p], p))[:n_sel]
                out[b, h, :len(order)] = sorted(order)
        return out


def reorder(table, lens, refs, parent, page: int, reserve=None):
    """(table, lens, refs, copies [(src, dst)], info) of b2_kv4_reorder, row by row."""
    bsz, most = table.shape
    new, length, left = np.full_like(table, -1), np.zeros_like(lens), refs.copy()
    for row in table:
        for p in row[row >= 0]:
            left[p] -= 1
    taken, wants = set(), []
    for b in range(bsz):
        par = int(parent[b])
        keep = 0
        if par >= 0:
            length[b] = lens[par]
            keep = most if par not in taken else int(lens[par]) // page
            new[b, :keep] = table[par, :keep]
        wants.append((par in taken and par >= 0 and lens[par] % page != 0, par))
        taken.add(par)
        for p in new[b][new[b] >= 0]:
            left[p] += 1
    free = [int(p) for p in np.flatnonzero(left == 0)]
    copies, missing = [], 0
    for b in range(bsz):
        more = int(reserve[b]) if reserve is not None else 0
        full, ntok = int(length[b]) // page, int(length[b]) + max(more, 0)
        want = -(-ntok // page)
        missing += max(0, want - most)
        for j in range(min(want, most)):
            if new[b, j] >= 0:
                continue
            copy = wants[b][0] and j == full
            if not free:
                missing += 1
                if copy:
                    length[b] = full * page
                continue
            new[b, j] = free.pop(0)
            left[new[b, j]] = 1
            if copy:
                copies.append((int(table[wants[b][1], full]), int(new[b, j])))
    return new, length, left, copies, np.array([(left == 0).sum(), len(copies), missing, 0], np.int32)


def compact(table, refs):
    """(table, refs, moves [(src, dst)], info) of b2_kv4_compact."""
    live = int((refs > 0).sum())
    holes = [p for p in range(live) if refs[p] <= 0]
    moved = [p for p in range(live, len(refs)) if refs[p] > 0]
    to = {p: p for p in range(live) if refs[p] > 0} | dict(zip(moved, holes))
    new = np.array([[to.get(int(p), -1) for p in row] for row in table], table.dtype)
    left = np.zeros_like(refs)
    for p, x in to.items():
        left[x] = refs[p]
    return new, left, list(zip(moved, holes)), np.array([live, len(moved), 0, 0], np.int32)
