"""The device's page table against one kept in lists: same ids, same bytes."""

import random

import pytest
import torch

from cxlsparse_b200 import CxsError
from cxlsparse_b200.pages import PageTable
from pages_case import PlainPages, caches_of, follow

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Pair:
    """A page table and its plain form, stepped together."""

    def __init__(self, layers, pages, kv_heads, dim, page_size, format, sequences, width):
        self.caches = caches_of(layers, pages, kv_heads, dim, page_size, format)
        self.table = PageTable(self.caches, sequences, width)
        self.plain = PlainPages(pages, sequences, width, page_size)
        self.codes = [c.codes.view(torch.uint8).clone() for c in self.caches]
        self.scales = [c.scales.clone() for c in self.caches]

    def step(self, name, *args):
        copies = getattr(self.plain, name)(*args)
        getattr(self.table, name)(*(ints(a) for a in args))
        if copies is None:
            with pytest.raises(CxsError):
                self.table.check()
        else:
            self.table.check()
            follow(copies, self.codes, self.scales)
        self.same()
        return copies

    def same(self):
        assert self.table.lengths.tolist() == self.plain.lengths
        assert torch.equal(self.table.table.cpu(), self.plain.table())
        assert self.table.references.tolist() == self.plain.references()
        for c, codes, scales in zip(self.caches, self.codes, self.scales):
            assert torch.equal(c.codes.view(torch.uint8), codes)
            assert torch.equal(c.scales, scales)


@pytest.mark.parametrize("layers,pages,kv_heads,dim,page_size,format,sequences,width", [
    (1, 40, 1, 64, 16, "e4m3", 1, 40), (3, 50, 2, 64, 64, "e4m3", 9, 7),
    (2, 300, 8, 128, 32, "int8", 40, 12), (16, 64, 2, 128, 16, "int8", 12, 33)])
def test_random_steps_follow_the_plain_table(cuda, layers, pages, kv_heads, dim, page_size, format,
                                             sequences, width):
    rng = random.Random(pages)
    pair = Pair(layers, pages, kv_heads, dim, page_size, format, sequences, width)
    did = dict.fromkeys(("extend", "fork", "free", "compact", "refused"), 0)
    for _ in range(60):
        empty = [b for b, n in enumerate(pair.plain.lengths) if n == 0]
        name = rng.choice(("extend", "extend", "fork", "fork", "free", "compact"))
        if name == "extend":
            args = [[rng.choice((0, 0, 1, 1, page_size, rng.randrange(3 * page_size)))
                     for _ in range(sequences)]]
        elif name == "fork":
            n = rng.randrange(1, len(empty) + 1) if empty else 1
            children = rng.sample(empty, n) if empty else [0]
            args = [[rng.randrange(sequences) for _ in children], children]
        elif name == "free":
            args = [[rng.randrange(sequences) for _ in range(rng.randrange(1, 4))]]
        else:
            args = []
        copies = pair.step(name, *args)
        did["refused" if copies is None else name] += 1
    assert did["extend"] and did["free"] and did["compact"]
    assert sequences == 1 or did["fork"]


def test_wrong_calls_change_nothing(cuda):
    pair = Pair(2, 6, 2, 64, 16, "e4m3", 5, 3)
    pair.step("extend", [20, 16, 0, 0, 0])                  # pages 0, 1 and 2
    for name, *args in (
            ("extend", [0, 33, 0, 0, 0]),                   # past the row
            ("extend", [0, -1, 5, 0, 0]),
            ("extend", [0, 0, 48, 1, 0]),                   # four pages of three
            ("fork", [0], [1]),                             # a child that holds tokens
            ("fork", [0, 0], [2, 2]),                       # twice
            ("fork", [0, 0, 5], [2, 3, 4]), ("fork", [0, -1], [2, 3]),
            ("fork", [0, 0], [2, 5]), ("fork", [0, 0], [2, -1]),
            ("fork", [0], [0])):
        assert pair.step(name, *args) is None
    pair.step("extend", [0, 32, 0, 0, 0])                   # one page is left
    assert pair.step("fork", [0, 0], [2, 3]) is None        # two are needed
    pair.step("fork", [0, 1, 4], [2, 3, 4])                 # an empty parent is its own child
    pair.step("free", [2, 2, 0, 2])
    pair.table.free(ints([7, 1, -1]))
    pair.plain.free([1])
    with pytest.raises(CxsError, match="out of range"):
        pair.table.check()
    pair.same()
    pair.table.free(ints([]))
    pair.table.fork(ints([]), ints([]))
    pair.same()


def test_adopted_tables(cuda):
    """Rows that share a partly filled page, entries past the lengths, pages and
    lengths out of range, a table narrower than the row."""
    pair = Pair(1, 20, 2, 64, 16, "int8", 4, 6)
    rows = [[7, 3, 11], [7, 3], [], [19]]
    wide = ints([[7, 3, 11, -5], [7, 3, 99, 2], [55, 1, 1, 1], [19, 0, 0, 0]])
    pair.table.adopt(wide[:, :3], ints([48, 20, 0, 16]))
    pair.plain.adopt(rows, [48, 20, 0, 16])
    pair.table.check()
    pair.same()
    assert pair.step("extend", [0, 1, 0, 0]) is None        # page 3 has two references
    pair.step("extend", [1, 0, 0, 1])
    pair.step("fork", [1], [2])
    pair.step("extend", [0, 0, 4, 0])                       # its own copy of page 3
    pair.step("free", [0])
    pair.step("extend", [0, 5, 0, 0])                       # and page 3 is the second row's
    pair.step("compact")
    # Its own tensors.
    pair.table.adopt(pair.table.table, pair.table.lengths)
    pair.same()
    pair.table.adopt(ints([[1, 20], [2, -3], [3, 4], [5, 6]]), ints([17, 17, 33, -1]))
    with pytest.raises(CxsError, match="page id outside the pool and lengths"):
        pair.table.check()
    assert pair.table.lengths.tolist() == [17, 17, 0, 0]
    assert pair.table.table[:, :2].tolist() == [[1, -1], [2, -1], [-1, -1], [-1, -1]]


@pytest.mark.parametrize("sequences", [1, 1025, 5000])
def test_many_sequences_and_pages(cuda, sequences):
    """More sequences than threads, a search through more pages than one round."""
    pages = 40000
    pair = Pair(1, pages, 1, 64, 16, "e4m3", sequences, 40000 // sequences)
    rng = random.Random(sequences)
    most = 30000 // sequences * 16
    pair.step("extend", [rng.randrange(most) for _ in range(sequences)])
    pair.step("free", [b for b in range(sequences) if rng.random() < 0.5] or [0])
    pair.step("extend", [rng.choice((0, 1, 17)) for _ in range(sequences)])
    pair.step("free", list(range(0, sequences, 3)))
    pair.step("fork", [1 % sequences] * len(range(0, sequences, 3)), list(range(0, sequences, 3)))
    assert pair.table.compact().item() == sum(r > 0 for r in pair.plain.references())
    follow(pair.plain.compact(), pair.codes, pair.scales)
    pair.same()


def test_captured_steps_and_another_stream(cuda):
    pair = Pair(2, 64, 2, 64, 16, "e4m3", 6, 8)
    pair.step("extend", [50, 33, 0, 0, 0, 0])
    children, parents, more = ints([2, 3, 4, 5]), ints([0, 1, 1, 0]), ints([1, 0, 3, 1, 0, 16])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        pair.table.free(children)
        pair.table.fork(parents, children)
        pair.table.extend(more)
    for _ in range(3):
        parents.copy_(ints([random.Random(_).randrange(2) for _ in range(4)]))
        graph.replay()
        pair.plain.free([2, 3, 4, 5])
        follow(pair.plain.fork(parents.tolist(), [2, 3, 4, 5]), pair.codes, pair.scales)
        pair.plain.extend(more.tolist())
        pair.table.check()
        pair.same()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pair.table.free(children)
        pair.table.compact()
    torch.cuda.current_stream().wait_stream(stream)
    pair.plain.free([2, 3, 4, 5])
    follow(pair.plain.compact(), pair.codes, pair.scales)
    pair.table.check()
    pair.same()
