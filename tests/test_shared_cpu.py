"""Refusals of attention over common tokens, without a device."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cxlsparse_b200 import _lib
from cxlsparse_b200.quantized import QuantizedCache

HEADER = Path(__file__).resolve().parent.parent / "include" / "cxlsparse.h"
P = 4096  # an address that is never followed


def shared_call(groups=P, shared=P, group_count=2, cache=None, **kw):
    held = dict(codes=P, scales=P, table=P, lengths=P, offsets=P, error=P, table_stride=4, pages=8,
                kv_heads=2, dim=64, page_size=64, format=0, users=200, width=4, tokens=200,
                max_tokens=2, type=0)
    held.update(cache or {})
    attend = dict(query=P, out=P, workspace=P, workspace_bytes=1 << 40, q_token_stride=2048,
                  q_head_stride=64, heads=32, scale=0.125)
    attend.update(kw)
    return _lib.CacheSharedCall(
        attend=_lib.CacheAttendCall(cache=_lib.CacheCall(**held), **attend), groups=groups,
        shared=shared, group_count=group_count)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc required")
def test_shared_struct_matches_c_layout(tmp_path):
    fields = [name for name, _ in _lib.CacheSharedCall._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "cxlsparse.h"',
             "int main(void) {"]
    lines += [f'printf("%zu\\n", offsetof(cxs_cache_shared_call, {f}));' for f in fields]
    lines += ['printf("%zu\\n", sizeof(cxs_cache_shared_call));', "return 0; }"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    want = [getattr(_lib.CacheSharedCall, f).offset for f in fields]
    assert [int(v) for v in out.stdout.split()] == want + [ctypes.sizeof(_lib.CacheSharedCall)]


@pytest.mark.parametrize("bad,status", [
    (dict(cache=dict(dim=32)), _lib.ERR_INVALID), (dict(cache=dict(type=2)), _lib.ERR_INVALID),
    (dict(cache=dict(users=70000)), _lib.ERR_CAPACITY), (dict(heads=3), _lib.ERR_INVALID),
    (dict(window=5), _lib.ERR_INVALID), (dict(group_count=-1), _lib.ERR_INVALID),
    (dict(group_count=201), _lib.ERR_INVALID), (dict(group_count=0), _lib.ERR_INVALID),
    (dict(cache=dict(tokens=1 << 26)), _lib.ERR_CAPACITY), (dict(groups=None), _lib.ERR_INVALID),
    (dict(shared=None), _lib.ERR_INVALID), (dict(query=None), _lib.ERR_INVALID),
    (dict(out=P + 8), _lib.ERR_INVALID), (dict(workspace=None), _lib.ERR_INVALID),
    (dict(workspace_bytes=1 << 10), _lib.ERR_INVALID), (dict(cache=dict(table=None)),
                                                        _lib.ERR_INVALID),
], ids=str)
def test_shared_refuses_before_any_launch(bad, status):
    lib = _lib.lib()
    assert lib.cxs_cache_attend_shared(shared_call(**bad), None) == status
    assert b"cache attend shared" in lib.cxs_last_error()


def test_workspace_grows_with_the_call():
    lib, size, more = _lib.lib(), _lib.c_i64(0), _lib.c_i64(0)
    assert lib.cxs_cache_attend_shared(None, None) == _lib.ERR_INVALID
    assert lib.cxs_cache_attend_shared_workspace(shared_call(), None) == _lib.ERR_INVALID
    assert lib.cxs_cache_attend_shared_workspace(shared_call(), size) == _lib.OK
    call = shared_call(cache=dict(tokens=4000, users=4000))
    assert lib.cxs_cache_attend_shared_workspace(call, more) == _lib.OK
    assert more.value > size.value > 0
    call = shared_call(cache=dict(tokens=0, max_tokens=0), query=None)
    assert lib.cxs_cache_attend_shared(call, None) == _lib.OK


def test_shared_arguments():
    cache = QuantizedCache(4, 2, 64, device="cpu")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)

    def ints(*v):
        return torch.tensor(v, dtype=torch.int32)

    table, lengths, offsets = torch.zeros(3, 2, dtype=torch.int32), ints(1, 1, 1), ints(0, 1, 2, 3)
    groups, shared = ints(0, 1, 3), ints(1, 1)
    good = dict(q=q, table=table, lengths=lengths, offsets=offsets, groups=groups, shared=shared)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(scale=math.nan), dict(table=table.long()),
                dict(lengths=lengths[:2]), dict(offsets=offsets[:3]), dict(groups=groups[:2]),
                dict(groups=groups.long()), dict(shared=shared.long()), dict(shared=shared[:1]),
                dict(shared=shared.view(1, 2)), dict(groups=ints(0, 0, 1, 2, 3), shared=ints(*[1] * 4)),
                dict(groups=ints(0), shared=ints()), dict(shared=ints(1, 1, 1, 1)[::2]),
                dict(max_tokens=-1), dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            cache.attend_shared(**{**good, **bad})
