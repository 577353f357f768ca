"""CPU restatement of the page operators: plain loops over Python lists."""

from __future__ import annotations

import torch


class PageState:
    """Tables, lengths, counts and the cache tensors ([lead, pages, segments,
    block, token bytes] uint8 each) of a paged cache."""

    def __init__(self, tables, lens, refs, caches, block):
        self.tables = [list(r) for r in tables]
        self.lens, self.refs, self.caches, self.block = list(lens), list(refs), caches, block

    def release(self, row, keep=0):
        for j in range(keep, len(self.tables[row])):
            if self.tables[row][j] >= 0:
                self.refs[self.tables[row][j]] -= 1
                self.tables[row][j] = -1

    def copy(self, src, dst, tokens):
        for c in self.caches:
            c[:, dst, :, :tokens] = c[:, src, :, :tokens]

    def copy_pages(self, src, dst):
        old = [c.clone() for c in self.caches]
        for i, (s, d) in enumerate(zip(src, dst)):
            pages = self.caches[0].shape[1]
            if not (0 <= s < pages and 0 <= d < pages) or dst.count(d) > 1 or d in src:
                continue
            for c, o in zip(self.caches, old):
                c[:, d] = o[:, s]

    def fork(self, src, dst):
        rows = len(self.tables)
        good = [0 <= s < rows and 0 <= d < rows for s, d in zip(src, dst)]
        named = [s for s, ok in zip(src, good) if ok]
        wanted = [d for d, ok in zip(dst, good) if ok]
        good = [ok and wanted.count(d) == 1 and d not in named for ok, d in zip(good, dst)]
        for d, ok in zip(dst, good):
            if ok:
                self.release(d)
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        out = []
        for s, d, ok in zip(src, dst, good):
            if not ok:
                out.append(-2)
                continue
            n = self.lens[s]
            full, tail = divmod(n, self.block)
            page = -1
            if tail:
                if not free:
                    out.append(-2)
                    self.lens[d] = 0
                    continue
                page = free.pop(0)
            for j in range(full):
                self.tables[d][j] = self.tables[s][j]
                self.refs[self.tables[s][j]] += 1
            if tail:
                self.tables[d][full] = page
                self.refs[page] = 1
                self.copy(self.tables[s][full], page, tail)
            self.lens[d] = n
            out.append(page)
        return out

    def free(self, rows, trim):
        for r in rows:
            if 0 <= r < len(self.tables):
                self.release(r, -(-self.lens[r] // self.block) if trim else 0)
                if not trim:
                    self.lens[r] = 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        to = dict(zip([p for p in live if p >= n], holes))
        for s, d in to.items():
            self.copy(s, d, self.block)
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.tables = [[to.get(p, p) for p in r] for r in self.tables]
        return n


def cache_bytes(t: torch.Tensor, page_dim: int) -> torch.Tensor:
    """A cache tensor as PageState holds it: values have one segment of
    [block, Hk * D] tokens a page, exponent bytes one per kv head."""
    lead = 1
    for s in t.shape[:page_dim]:
        lead *= s
    pages, page = t.shape[page_dim], t.shape[page_dim + 1:]
    raw = t.contiguous().view(torch.uint8)
    if len(page) == 3:
        return raw.reshape(lead, pages, 1, page[0], -1)
    return raw.reshape(lead, pages, page[0], page[1], -1)
