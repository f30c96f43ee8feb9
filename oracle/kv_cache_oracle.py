"""CPU oracle of the paged KV cache: new rows into their pages, and the pages' bookkeeping.

TEST INFRASTRUCTURE ONLY: imported by ``tests/`` as the oracle of the HIP kernels, never by the product.

``store`` follows nanoserve/model/rope.py:78-91 (rotate-half) and nanoserve/model/attention.py:55-72 (the write) in
float64, one token after the other; a token's position is the one of oracle/paged_attention_oracle.py.  ``Pool``
restates the page operators' contracts with Python loops over plain lists.
"""
from __future__ import annotations

import math

import numpy as np


def store(query, key, value, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens, block_size,
          inv_freq=None):
    """float64 (rotated query or None, k_cache, v_cache) after the call, and the bound's scale |x| + |y| of each
    rotated element in arrays alike (0 where nothing is computed)."""
    out = None if query is None else np.array(query, dtype=np.float64)
    k, v = np.array(k_cache, dtype=np.float64), np.array(v_cache, dtype=np.float64)
    s_q = None if query is None else np.zeros(out.shape)
    s_k = np.zeros(k.shape)
    half = key.shape[2] // 2

    def turned(x, pos):
        a = pos * np.asarray(inv_freq, dtype=np.float64)
        lo, hi = x[..., :half], x[..., half:]
        y = np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], axis=-1)
        return y, np.concatenate([np.abs(lo) + np.abs(hi)] * 2, axis=-1)

    for s in range(len(seq_lens)):
        for n in range(int(query_lens[s])):
            i = int(query_start_loc[s]) + n
            pos = int(seq_lens[s]) - int(query_lens[s]) + n
            if i >= key.shape[0] or pos < 0:
                continue
            col = pos // block_size
            page = int(block_tables[s][col]) if col < block_tables.shape[1] else -1
            row = np.asarray(key[i], dtype=np.float64)
            scale = 0.0
            if inv_freq is not None:
                row, scale = turned(row, pos)
                if out is not None:
                    out[i], s_q[i] = turned(np.asarray(query[i], dtype=np.float64), pos)
            if 0 <= page < k.shape[0]:
                k[page, pos % block_size], s_k[page, pos % block_size] = row, scale
                v[page, pos % block_size] = value[i]
    return out, k, v, s_q, s_k


class Pool:
    """Tables, lengths, counts and page contents (any array of pages) of a pool, changed in place."""

    NO_PAGES, BAD_ROW, BAD_LENGTH = 2, 4, 8

    def __init__(self, tables, lens, refs, block_size, pages):
        self.tables, self.lens, self.refs = np.array(tables), np.array(lens), np.array(refs)
        self.bs, self.pages, self.status = block_size, np.array(pages), 0   # pages: (page, slot, ...)

    def _free_pages(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def _first_listings(self, rows):
        seen, ok = set(), []
        for r in rows:
            ok.append(0 <= r < len(self.lens) and r not in seen)
            seen.add(r)
            if not ok[-1]:
                self.status |= self.BAD_ROW
        return ok

    def extend(self, rows, lens):
        free, asked = self._free_pages(), 0
        for r, n, ok in zip(rows, lens, self._first_listings(rows)):
            if not ok:
                continue
            if n < self.lens[r] or n > self.tables.shape[1] * self.bs:
                self.status |= self.BAD_LENGTH
                continue
            a, b = -(-int(self.lens[r]) // self.bs), -(-int(n) // self.bs)
            asked += b - a
            if b > a and asked > len(free):
                self.status |= self.NO_PAGES
                continue
            for j in range(a, b):
                p = free[asked - (b - a) + j - a]
                self.tables[r, j], self.refs[p] = p, 1
            self.lens[r] = n

    def fork(self, parents, children):
        free, asked = self._free_pages(), 0
        was = self.lens.copy()
        for a, c, ok in zip(parents, children, self._first_listings(children)):
            if not ok or not 0 <= a < len(was) or was[c] != 0:
                self.status |= self.BAD_ROW
                continue
            n = int(was[a])
            cols = -(-n // self.bs)
            row = self.tables[a, :cols].copy()
            if n % self.bs and row[-1] >= 0:
                asked += 1
                if asked > len(free):
                    self.status |= self.NO_PAGES
                    continue
                p = free[asked - 1]
                self.pages[p, :n % self.bs] = self.pages[row[-1], :n % self.bs]
                row[-1] = p
            for p in row[row >= 0]:
                self.refs[p] += 1
            self.tables[c, :cols], self.lens[c] = row, n

    def free(self, rows):
        for r in rows:
            if not 0 <= r < len(self.lens):
                self.status |= self.BAD_ROW
                continue
            self._drop(r, 0, -(-int(self.lens[r]) // self.bs))
            self.lens[r] = 0

    def release(self, rows, window, sinks):
        for r in rows:
            if not 0 <= r < len(self.lens):
                self.status |= self.BAD_ROW
                continue
            gone = int(self.lens[r]) - window + 1
            self._drop(r, -(-sinks // self.bs), max(0, math.floor(gone / self.bs)))

    def _drop(self, r, first, last):
        for j in range(first, min(last, -(-int(self.lens[r]) // self.bs))):
            if self.tables[r, j] >= 0:
                self.refs[self.tables[r, j]] -= 1
                self.tables[r, j] = -1

    def compact(self):
        """The page map, and the pool compacted in place."""
        used = [p for p in range(len(self.refs)) if self.refs[p] != 0]
        m = len(used)
        holes = [p for p in range(m) if self.refs[p] == 0]
        page_map = np.full(len(self.refs), -1)
        for p in used:
            to = p if p < m else holes.pop(0)
            page_map[p] = to
            if to != p:
                self.pages[to] = self.pages[p]
                self.refs[to], self.refs[p] = self.refs[p], 0
        for r in range(len(self.lens)):
            for j in range(-(-int(self.lens[r]) // self.bs)):
                if self.tables[r, j] >= 0:
                    self.tables[r, j] = page_map[self.tables[r, j]]
        return page_map
