"""Refusals of the page table, without a device."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cxlsparse_b200 import _lib
from cxlsparse_b200.pages import PageTable
from cxlsparse_b200.quantized import QuantizedCache

HEADER = Path(__file__).resolve().parent.parent / "include" / "cxlsparse.h"
P = 4096  # an address that is never followed


def pages_call(**kw):
    base = dict(layer_buffers=P, table=P, lengths=P, references=P, lowest=P, error=P, workspace=P,
                workspace_bytes=1 << 30, layers=2, pages=8, kv_heads=2, dim=64, page_size=64,
                sequences=3, width=4)
    base.update(kw)
    return _lib.PagesCall(**base)


def calls(lib, call):
    return [lib.cxs_pages_extend(call, P, None), lib.cxs_pages_fork(call, P, P, 2, None),
            lib.cxs_pages_free(call, P, 2, None), lib.cxs_pages_adopt(call, P, 4, 4, P, None),
            lib.cxs_pages_compact(call, P, None)]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc required")
def test_pages_struct_matches_c_layout(tmp_path):
    fields = [name for name, _ in _lib.PagesCall._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "cxlsparse.h"',
             "int main(void) {"]
    lines += [f'printf("%zu\\n", offsetof(cxs_pages_call, {f}));' for f in fields]
    lines += ['printf("%zu\\n", sizeof(cxs_pages_call));', "return 0; }"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    want = [getattr(_lib.PagesCall, f).offset for f in fields] + [ctypes.sizeof(_lib.PagesCall)]
    assert [int(v) for v in out.stdout.split()] == want


@pytest.mark.parametrize("bad,status", [
    (dict(pages=0), _lib.ERR_INVALID), (dict(layers=0), _lib.ERR_INVALID),
    (dict(sequences=0), _lib.ERR_INVALID), (dict(width=0), _lib.ERR_INVALID),
    (dict(kv_heads=0), _lib.ERR_INVALID), (dict(dim=96), _lib.ERR_INVALID),
    (dict(page_size=48), _lib.ERR_INVALID), (dict(table=None), _lib.ERR_INVALID),
    (dict(lengths=None), _lib.ERR_INVALID), (dict(references=None), _lib.ERR_INVALID),
    (dict(lowest=None), _lib.ERR_INVALID), (dict(layer_buffers=None), _lib.ERR_INVALID),
    (dict(workspace=None), _lib.ERR_INVALID), (dict(workspace_bytes=16), _lib.ERR_INVALID),
    (dict(workspace=P + 2), _lib.ERR_INVALID), (dict(width=1 << 25), _lib.ERR_CAPACITY),
    (dict(width=1 << 20, sequences=1 << 12), _lib.ERR_CAPACITY),
], ids=str)
def test_pages_calls_refuse_before_any_launch(bad, status):
    lib = _lib.lib()
    assert calls(lib, pages_call(**bad)) == [status] * 5
    assert b"pages compact" in lib.cxs_last_error()


def test_pages_arguments_are_refused():
    lib = _lib.lib()
    call, size = pages_call(), _lib.c_i64(0)
    assert calls(lib, None) == [_lib.ERR_INVALID] * 5
    assert lib.cxs_pages_workspace(call, None) == _lib.ERR_INVALID
    assert lib.cxs_pages_workspace(call, size) == _lib.OK and size.value > 0
    assert lib.cxs_pages_fork(call, P, P, 4, None) == _lib.ERR_INVALID
    assert lib.cxs_pages_fork(call, P, P, -1, None) == _lib.ERR_INVALID
    assert lib.cxs_pages_fork(call, None, P, 2, None) == _lib.ERR_INVALID
    assert lib.cxs_pages_fork(call, None, None, 0, None) == _lib.OK
    assert lib.cxs_pages_free(call, None, 2, None) == _lib.ERR_INVALID
    assert lib.cxs_pages_free(call, P, -2, None) == _lib.ERR_INVALID
    assert lib.cxs_pages_free(call, None, 0, None) == _lib.OK
    for table, stride, width, lengths in ((None, 4, 4, P), (P, 4, 4, None), (P, 4, 5, P),
                                          (P, 3, 4, P), (P, 4, 0, P)):
        assert lib.cxs_pages_adopt(call, table, stride, width, lengths, None) == _lib.ERR_INVALID


def test_page_table_refusals():
    def cache(*args, **kw):
        return QuantizedCache(*args, device="cpu", **kw)

    a, b = cache(4, 2, 64), cache(4, 2, 64)
    table = PageTable([a, b], 3, 5)
    assert table.table.shape == (3, 5) and (table.table == -1).all()
    assert table.lengths.tolist() == [0] * 3 and table.references.tolist() == [0] * 4
    for caches, sequences, width in (
            ([], 3, 5), ([a, a], 3, 5), ([a, cache(5, 2, 64)], 3, 5), ([a, "b"], 3, 5),
            ([a, cache(4, 2, 128)], 3, 5), ([a, cache(4, 2, 64, page_size=32)], 3, 5),
            ([a, cache(4, 2, 64, format="int8")], 3, 5), ([a], 0, 5), ([a], 3, 0)):
        with pytest.raises(ValueError):
            PageTable(caches, sequences, width)
    ints = torch.zeros(3, dtype=torch.int32)
    wide = torch.zeros(3, 6, dtype=torch.int32)
    for call, args in (
            (table.extend, (ints[:2],)), (table.extend, (ints.long(),)),
            (table.extend, (torch.zeros(6, dtype=torch.int32)[::2],)),
            (table.fork, (ints, ints[:2])), (table.fork, (ints.long(), ints)),
            (table.fork, (torch.zeros(4, dtype=torch.int32),) * 2),
            (table.fork, (ints, ints.view(1, 3))), (table.free, (ints.float(),)),
            (table.free, (wide,)), (table.adopt, (wide, ints)),
            (table.adopt, (wide[:2, :5], ints)), (table.adopt, (wide[:, :5].long(), ints)),
            (table.adopt, (wide[:, :5], ints[:2])), (table.adopt, (wide[:, :0], ints)),
            (table.adopt, (wide.t()[:3], ints)), (table.adopt, (wide[:1, :5].expand(3, 5), ints))):
        with pytest.raises(ValueError):
            call(*args)
