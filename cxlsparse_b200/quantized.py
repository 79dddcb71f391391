"""Dense 8-bit key/value cache in HBM over the C ABI (``cxs_cache_*``).

The selected-block path keeps a user's history in 16 bits in the host pool. A
``QuantizedCache`` keeps one layer's whole histories in HBM at 8 bits a
channel, in pages with a scale for each page, KV head and part (K or V):

- ``append`` quantises new tokens into the pages as they arrive;
- ``read`` brings tokens back to 16 or 32 bits;
- ``attend`` is dense attention of new tokens' queries over them (one token a
  user, a suffix, or a prefill chunk).

The three take the same description of a step: ``table [users, width]`` int32
page ids (shared by all layers of a model), ``lengths [users]`` int32 tokens
with the new ones counted, and ``offsets [users + 1]`` int32, the packed rows
of each user (None: one new token for every user). No gradient passes through
them. No counterpart in the reference.
"""

import math
import threading

import torch

from . import _lib

FORMATS = {"e4m3": 0, "int8": 1}
CODE_TYPES = {torch.float8_e4m3fn: 0, torch.int8: 1}
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class QuantizedCache:
    """One layer's pages: ``codes [pages, kv_heads, 2, page_size, dim]``
    (float8_e4m3fn or int8) and ``scales [pages, kv_heads, 2]`` fp32; a value
    is code * scale. Give the sizes for a new cache, or both tensors."""

    def __init__(self, pages=None, kv_heads=None, dim=None, *, page_size=64, format="e4m3",
                 device="cuda", codes=None, scales=None):
        if (codes is None) != (scales is None):
            raise ValueError("codes and scales come together")
        if codes is None:
            if format not in FORMATS:
                raise ValueError(f"unknown cache format {format!r}")
            dtype = {v: k for k, v in CODE_TYPES.items()}[FORMATS[format]]
            if dim not in (64, 128) or page_size not in (16, 32, 64):
                raise ValueError("dim must be 64 or 128, page_size 16, 32 or 64")
            if not pages or pages < 1 or not kv_heads or kv_heads < 1:
                raise ValueError("pages and kv_heads must be positive")
            codes = torch.zeros((pages, kv_heads, 2, page_size, dim), dtype=torch.uint8,
                                device=device).view(dtype)
            scales = torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=device)
        if codes.ndim != 5 or codes.shape[2] != 2 or codes.dtype not in CODE_TYPES:
            raise ValueError("codes must be [pages, kv_heads, 2, page_size, dim] in "
                             "float8_e4m3fn or int8")
        if codes.shape[3] not in (16, 32, 64) or codes.shape[4] not in (64, 128):
            raise ValueError("page_size must be 16, 32 or 64 and dim 64 or 128")
        if scales.shape != codes.shape[:3] or scales.dtype != torch.float32:
            raise ValueError("scales must be [pages, kv_heads, 2] fp32")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        if scales.device != codes.device:
            raise ValueError("codes and scales must be on one device")
        self.codes, self.scales = codes, scales
        self.pages, self.kv_heads, _, self.page_size, self.dim = codes.shape
        self.format = CODE_TYPES[codes.dtype]
        self.device = codes.device
        self.error = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._first = torch.zeros(1, dtype=torch.int64, device=self.device)
        self._lock = threading.Lock()
        self._codes, self._scales, self._error = (
            t.data_ptr() for t in (codes, scales, self.error))
        self._workspace = {}

    # -- checks ------------------------------------------------------------
    def check(self):
        """Wait for the device, the calls on all its streams, and raise if one
        met a page or length out of range since the last check (such tokens are
        skipped, never followed), or gave up a wait."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        with self._lock:
            bits = int(self.error.item())
            if bits:
                # Taken off by an atomic addition: bits that a call of another
                # thread sets meanwhile stay for the next check.
                self.error.index_add_(0, self._first, torch.full_like(self.error, -bits))
        if bits:
            what = [text for bit, text in (
                (_lib.DEVICE_ERR_BAD_BLOCK, "a page id outside the cache"),
                (_lib.DEVICE_ERR_BAD_LENGTH, "lengths or offsets out of range"),
                (_lib.DEVICE_ERR_COPY_TIMEOUT, "a wait inside the kernel that ran out (its "
                 "result is not valid)")) if bits & bit]
            raise _lib.CxsError(_lib.ERR_INVALID, "cache call met " + " and ".join(what))

    def _call(self, table, lengths, offsets, tokens, max_tokens, type_):
        """The fields of ``cxs_cache_call``."""
        shape, stride = table.shape, table.stride()
        if len(shape) != 2 or table.dtype != torch.int32 or stride[1] != 1:
            raise ValueError("table must be [users, width] int32 with contiguous rows")
        users, width = shape
        if lengths.shape != (users,) or lengths.dtype != torch.int32 \
                or not lengths.is_contiguous():
            raise ValueError("lengths must be [users] int32, contiguous")
        if table.device != self.device or lengths.device != self.device:
            raise ValueError(f"table and lengths must be on {self.device}")
        if offsets is None:
            if tokens != users:
                raise ValueError("without offsets every user has one row")
            at, most = 0, 1
        else:
            if offsets.shape != (users + 1,) or offsets.dtype != torch.int32 \
                    or not offsets.is_contiguous() or offsets.device != self.device:
                raise ValueError(f"offsets must be [users + 1] int32, contiguous, on {self.device}")
            at, most = offsets.data_ptr(), tokens
        if max_tokens is not None:
            if max_tokens < 0:
                raise ValueError("max_tokens must not be negative")
            most = min(most, max_tokens)
        return (self._codes, self._scales, table.data_ptr(), lengths.data_ptr(), at, self._error,
                stride[0], self.pages, self.kv_heads, self.dim, self.page_size, self.format,
                users, width, tokens, most, type_)

    def _rows(self, name, x):
        """(shape, strides) of a [tokens, heads, dim] tensor."""
        shape, stride = x.shape, x.stride()
        if len(shape) != 3 or shape[2] != self.dim or stride[2] != 1:
            raise ValueError(f"{name} must be [tokens, heads, {self.dim}] with contiguous channels")
        if x.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        return shape, stride

    def _queries(self, q, scale):
        """(tokens, heads, strides, scale) of an attend call's queries."""
        shape, stride = self._rows("q", q)
        if q.requires_grad and torch.is_grad_enabled():
            raise ValueError("the cache has no gradient: attend with a detached q")
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("q must be bf16 or fp16")
        if shape[1] < 1 or shape[1] % self.kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        scale = self.dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        return shape[0], shape[1], stride, scale

    def _workspace_size(self, known, fn, call):
        """Scratch of an attend call, kept by what it depends on."""
        size = _lib.c_i64(0)
        _lib.check(fn(call, size))
        if len(self._workspace) >= 4096:
            self._workspace.clear()
        self._workspace[known] = size.value
        return size.value

    # -- operators ---------------------------------------------------------
    def append(self, k, v, table, lengths, offsets=None, *, max_tokens=None):
        """Quantise the new tokens' keys and values [tokens, kv_heads, dim]
        (bf16, fp16 or fp32) into their pages. ``max_tokens``: most new tokens
        of one user, if known on the host (it bounds the launch; a user with
        more is left as it was, with an error that ``check`` raises)."""
        (shape, ks), (v_shape, vs) = self._rows("k", k), self._rows("v", v)
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            raise ValueError("the cache has no gradient: append detached k and v")
        if shape[1] != self.kv_heads or v_shape != shape:
            raise ValueError(f"k and v must both be [tokens, {self.kv_heads}, {self.dim}]")
        dtype = k.dtype
        if dtype not in TYPES or v.dtype != dtype:
            raise ValueError("k and v must be bf16, fp16 or fp32, of one type")
        call = _lib.pack_cache_call(
            *self._call(table, lengths, offsets, shape[0], max_tokens, TYPES[dtype]))
        _lib.on_device(self.device.index, _lib.packed().cxs_cache_append, call, k.data_ptr(),
                       ks[0], ks[1], v.data_ptr(), vs[0], vs[1])

    def read(self, table, starts, offsets, *, total, max_tokens=None, dtype=torch.bfloat16):
        """``(k, v)`` [total, kv_heads, dim] of consecutive tokens: row
        offsets[b] + i is user b's token starts[b] + i, and rows that no user
        has are 0."""
        if dtype not in TYPES:
            raise ValueError("dtype must be bf16, fp16 or fp32")
        call = _lib.pack_cache_call(
            *self._call(table, starts, offsets, total, max_tokens, TYPES[dtype]))
        k = torch.empty((total, self.kv_heads, self.dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _lib.on_device(self.device.index, _lib.packed().cxs_cache_read, call, k.data_ptr(),
                       v.data_ptr())
        return k, v

    def attend(self, q, table, lengths, offsets=None, *, max_tokens=None, causal=True, window=0,
               scale=None, return_lse=False):
        """Attention of queries [tokens, heads, dim] (bf16 or fp16) over the
        cached tokens of their users, which include the new ones: append first.
        The last of user b's rows is at position lengths[b] - 1. ``window``: a
        row also sees only the last ``window`` positions up to its own. Returns
        [tokens, heads, dim], with ``return_lse`` also the softmax's log-sum
        [tokens, heads] fp32 (for joining with attention over other keys)."""
        tokens, heads, stride, scale = self._queries(q, scale)
        if window < 0:
            raise ValueError("window must not be negative")
        common = self._call(table, lengths, offsets, tokens, max_tokens, TYPES[q.dtype])
        size = self._workspace.get((heads, common[15]))
        if size is None:
            size = self._workspace_size(
                (heads, common[15]), _lib.packed().cxs_cache_attend_workspace,
                _lib.pack_cache_attend_call(*common, 0, 0, 0, 0, 0, 0, 0, heads, 1, 0, 1.0))
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=self.device) \
            if return_lse else None
        workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
        call = _lib.pack_cache_attend_call(
            *common, q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            workspace.data_ptr(), size, stride[0], stride[1], heads, bool(causal), window, scale)
        _lib.on_device(self.device.index, _lib.packed().cxs_cache_attend, call)
        return (out, lse) if return_lse else out

    def attend_shared(self, q, table, lengths, offsets, groups, shared, *, max_tokens=None,
                      causal=True, scale=None, return_lse=False):
        """``attend`` for users that have their first tokens in common, such as
        the candidates of one history (``PageTable.fork``): the common tokens are
        read once for all of them. Users groups[g] .. groups[g + 1] - 1 (``groups
        [count + 1]`` int32, ascending from 0 to all users) are group g; their
        first shared[g] tokens (``shared [count]`` int32) are the same, codes and
        scales, in whichever pages. A user alone is a group of its own, with 0
        shared tokens if need be; one without rows may hold other tokens, or none.
        Groups that do not ascend are an error that ``check`` raises (rows are
        0); calls with few rows are computed user by user and do not look at
        them."""
        tokens, heads, stride, scale = self._queries(q, scale)
        common = self._call(table, lengths, offsets, tokens, max_tokens, TYPES[q.dtype])
        users, count = common[12], shared.shape[0] if shared.ndim == 1 else -1
        for name, x, n in (("shared", shared, count), ("groups", groups, count + 1)):
            if x.shape != (n,) or x.dtype != torch.int32 or not x.is_contiguous() \
                    or x.device != self.device:
                raise ValueError("shared must be [groups] and groups [groups + 1] int32, "
                                 f"contiguous, on {self.device}")
        if count > users or (tokens and not count):
            raise ValueError("every group must have a user, every row a group")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=self.device) \
            if return_lse else None
        known = heads, common[15], tokens, users, count
        size = self._workspace.get(known)
        if size is None:
            size = self._workspace_size(
                known, _lib.packed().cxs_cache_attend_shared_workspace,
                _lib.pack_cache_shared_call(*common, 0, 0, 0, 0, 0, 0, 0, heads, 1, 0, 1.0, 0, 0,
                                            count))
        workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
        call = _lib.pack_cache_shared_call(
            *common, q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            workspace.data_ptr(), size, stride[0], stride[1], heads, bool(causal), 0, scale,
            groups.data_ptr(), shared.data_ptr(), count)
        _lib.on_device(self.device.index, _lib.packed().cxs_cache_attend_shared, call)
        return (out, lse) if return_lse else out
