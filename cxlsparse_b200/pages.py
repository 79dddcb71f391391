"""Sequences over the pages of the dense 8-bit cache, kept on the device
(``cxs_pages_*``).

``QuantizedCache`` takes page tables as they come. A ``PageTable`` keeps one for
all layers of a model and changes it without the host: room for new tokens,
several continuations of one history (``fork`` shares its full pages and copies
the partly filled one), sequences that end, a pool brought together. Its
``table`` and ``lengths`` are what ``append``, ``attend``, ``attend_shared`` and
``read`` take, so a decode step with all of them can be captured in a CUDA
graph. No counterpart in the reference.
"""

import torch

from . import _lib
from .quantized import QuantizedCache


class PageTable:
    """``table [sequences, width]`` int32 page ids (-1: none), ``lengths
    [sequences]`` and ``references [pages]`` (table entries that name a page)
    over ``caches``, the layers' ``QuantizedCache`` of one shape. All sequences
    are empty at first. A page id is one page of every layer.

    Pages are handed out lowest id first in the order of the sequences, so a
    run gives the same table every time. Calls change the state in place and
    must follow one another (on one stream, or ordered between streams)."""

    def __init__(self, caches, sequences, width):
        caches = list(caches)
        if not caches or not all(isinstance(c, QuantizedCache) for c in caches):
            raise ValueError("caches must be the layers' QuantizedCache")
        first = caches[0]
        for c in caches:
            if c.codes.shape != first.codes.shape or c.device != first.device \
                    or c.format != first.format:
                raise ValueError("the layers' caches must agree in shape, format and device")
        if len({c.codes.data_ptr() for c in caches}) < len(caches):
            raise ValueError("a cache is there twice")
        if sequences < 1 or width < 1:
            raise ValueError("sequences and width must be positive")
        self.caches, self.device = caches, first.device
        self.sequences, self.width, self.pages = sequences, width, first.pages
        self.page_size = first.page_size

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device=self.device)

        self.table = ints(sequences, width, fill=-1)
        self.lengths = ints(sequences)
        self._references = ints(self.pages + 1)  # and the lowest page that may be free
        self.references = self._references[:self.pages]
        self.error = ints(1)
        self._first = torch.zeros(1, dtype=torch.int64, device=self.device)
        self._buffers = torch.tensor([[c.codes.data_ptr(), c.scales.data_ptr()] for c in caches],
                                     dtype=torch.int64, device=self.device)

        def call(workspace, size):
            return _lib.pack_pages_call(
                self._buffers.data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(),
                self.references.data_ptr(), self._references[self.pages:].data_ptr(),
                self.error.data_ptr(), workspace, size, len(caches), self.pages, first.kv_heads,
                first.dim, first.page_size, sequences, width)

        size = _lib.c_i64(0)
        _lib.check(_lib.packed().cxs_pages_workspace(call(0, 0), size))
        self._workspace = ints(size.value // 4)
        self._call = call(self._workspace.data_ptr(), size.value)

    def _ids(self, name, x, shape=None):
        if x.dtype != torch.int32 or x.ndim != 1 or not x.is_contiguous() \
                or x.device != self.device or (shape is not None and x.shape != shape):
            raise ValueError(f"{name} must be int32, contiguous, of one dimension"
                             + (f" and {shape[0]} entries" if shape else "")
                             + f", on {self.device}")
        return x.data_ptr()

    def _run(self, fn, *args):
        _lib.on_device(self.device.index, fn, self._call, *args)

    # -- operators ---------------------------------------------------------
    def extend(self, counts=None):
        """Room for ``counts [sequences]`` int32 more tokens of each sequence
        (None: one each): ``lengths`` grow by them and rows get the pages they
        need. Nothing changes, with an error that ``check`` raises, where pages
        or a row do not suffice, or where tokens would go on in a page that
        another row names too (only ``adopt`` brings such rows: fork them)."""
        at = 0 if counts is None else self._ids("counts", counts, self.lengths.shape)
        self._run(_lib.packed().cxs_pages_extend, at)

    def fork(self, parents, children):
        """Sequences ``children [n]``, empty before, become copies of ``parents
        [n]`` (int32): full pages are shared, of a partly filled last page each
        child gets its own copy, in every layer. A parent may be there often, a
        child once; otherwise, or where pages do not suffice, nothing changes,
        with an error that ``check`` raises."""
        at = self._ids("parents", parents)
        to = self._ids("children", children, parents.shape)
        if len(parents) > self.sequences:
            raise ValueError("more children than sequences")
        self._run(_lib.packed().cxs_pages_fork, at, to, len(parents))

    def free(self, sequences):
        """The sequences (int32 ids) hold nothing any more; their pages are free
        but for those that others share."""
        at = self._ids("sequences", sequences)
        self._run(_lib.packed().cxs_pages_free, at, len(sequences))

    def adopt(self, table, lengths):
        """Take over ``table [sequences, at most width]`` and ``lengths
        [sequences]`` (int32) in the place of what the sequences held. Rows may
        share pages. Page ids outside the pool become -1, and a length outside
        its row 0, with an error that ``check`` raises."""
        at = self._ids("lengths", lengths, self.lengths.shape)
        shape, stride = table.shape, table.stride()
        if len(shape) != 2 or shape[0] != self.sequences or not 1 <= shape[1] <= self.width \
                or table.dtype != torch.int32 or stride[1] != 1 or table.device != self.device:
            raise ValueError(f"table must be [{self.sequences}, at most {self.width}] int32 with "
                             f"contiguous rows, on {self.device}")
        # (The rows of a table of one sequence have no distance.)
        stride = stride[0] if self.sequences > 1 else shape[1]
        if stride < shape[1]:
            raise ValueError("the table's rows overlap")
        self._run(_lib.packed().cxs_pages_adopt, table.data_ptr(), stride, shape[1], at)

    def compact(self):
        """Move pages, in every layer, until the n pages in use are the first n;
        returns n as an int32 tensor [1]. The rest of the pool holds nothing."""
        live = self.lengths.new_empty(1)
        self._run(_lib.packed().cxs_pages_compact, live.data_ptr())
        return live

    def check(self):
        """Wait for the device and raise if a call met something wrong since the
        last check."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        bits = int(self.error.item())
        if bits:
            # (An atomic addition: bits that a call sets meanwhile stay.)
            self.error.index_add_(0, self._first, torch.full_like(self.error, -bits))
            what = [text for bit, text in (
                (_lib.DEVICE_ERR_NO_PAGES, "too few free pages (nothing was changed)"),
                (_lib.DEVICE_ERR_BAD_SEQUENCE, "a sequence out of range, or a child that holds "
                 "tokens or is there twice"),
                (_lib.DEVICE_ERR_SHARED_PAGE, "new tokens for a page with other references "
                 "(nothing was changed)"),
                (_lib.DEVICE_ERR_BAD_BLOCK, "a page id outside the pool"),
                (_lib.DEVICE_ERR_BAD_LENGTH, "lengths or counts outside the row")) if bits & bit]
            raise _lib.CxsError(_lib.ERR_INVALID, "page table call met " + " and ".join(what))
