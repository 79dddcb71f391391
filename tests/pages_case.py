"""A page table kept in lists, and caches whose bytes tell where they came from."""

import torch

from cxlsparse_b200.quantized import QuantizedCache


class PlainPages:
    """What ``PageTable`` does, page by page. Calls return the copies they make
    as (source page, target page, slots), or None where nothing changes."""

    def __init__(self, pages, sequences, width, page_size):
        self.pages, self.width, self.page_size = pages, width, page_size
        self.rows = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences

    def references(self):
        found = [0] * self.pages
        for row in self.rows:
            for p in row:
                found[p] += 1
        return found

    def _free(self, n):
        free = [p for p, r in enumerate(self.references()) if r == 0]
        return free[:n] if len(free) >= n else None

    def extend(self, counts):
        need, uses = [], self.references()
        for row, length, n in zip(self.rows, self.lengths, counts):
            if n < 0 or length + n > self.width * self.page_size:
                return None
            if n and length % self.page_size and uses[row[-1]] > 1:
                return None
            need.append(-(-(length + n) // self.page_size) - len(row))
        fresh = self._free(sum(need))
        if fresh is None:
            return None
        for b, n in enumerate(need):
            self.rows[b] += fresh[:n]
            del fresh[:n]
            self.lengths[b] += counts[b]
        return []

    def fork(self, parents, children):
        n = len(self.rows)
        if any(not 0 <= x < n for x in parents + children) or len(set(children)) < len(children) \
                or any(self.lengths[c] for c in children):
            return None
        sizes = [self.lengths[p] for p in parents]
        fresh = self._free(sum(s % self.page_size > 0 for s in sizes))
        if fresh is None:
            return None
        copies = []
        for parent, child, size in zip(parents, children, sizes):
            full = size // self.page_size
            row = self.rows[parent][:full]
            if size % self.page_size:
                copies.append((self.rows[parent][full], fresh.pop(0), size % self.page_size))
                row = row + [copies[-1][1]]
            self.rows[child], self.lengths[child] = row, size
        return copies

    def free(self, sequences):
        for b in sequences:
            if 0 <= b < len(self.rows):
                self.rows[b], self.lengths[b] = [], 0
        return []

    def adopt(self, rows, lengths):
        self.rows, self.lengths = [list(r) for r in rows], list(lengths)
        return []

    def compact(self):
        uses = self.references()
        live = sum(r > 0 for r in uses)
        holes = [p for p in range(live) if not uses[p]]
        names = dict(zip([p for p in range(live, self.pages) if uses[p]], holes))
        self.rows = [[names.get(p, p) for p in row] for row in self.rows]
        return [(s, t, self.page_size) for s, t in names.items()]

    def table(self):
        return torch.tensor([r + [-1] * (self.width - len(r)) for r in self.rows],
                            dtype=torch.int32)


def caches_of(layers, pages, kv_heads, dim, page_size, format, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    made = []
    for _ in range(layers):
        c = QuantizedCache(pages, kv_heads, dim, page_size=page_size, format=format)
        c.codes.view(torch.uint8).copy_(torch.randint(0, 256, c.codes.shape, generator=g,
                                                      device="cuda", dtype=torch.uint8))
        c.scales.copy_(torch.rand(c.scales.shape, generator=g, device="cuda"))
        made.append(c)
    return made


def follow(copies, codes, scales):
    """The copies, on plain tensors of every layer."""
    for c, s in zip(codes, scales):
        old_c, old_s = c.clone(), s.clone()
        for source, target, slots in copies:
            c[target, :, :, :slots] = old_c[source, :, :, :slots]
            s[target] = old_s[source]
