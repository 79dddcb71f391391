"""Refusals and host logic of the dense 8-bit cache and the rotary positions,
without a device."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cxlsparse_b200 import _lib
from cxlsparse_b200.quantized import QuantizedCache
from cxlsparse_b200.rotary import Rotary, frequencies

HEADER = Path(__file__).resolve().parent.parent / "include" / "cxlsparse.h"
P = 4096  # an address that is never followed


def cache_call(**kw):
    base = dict(codes=P, scales=P, table=P, lengths=P, offsets=P, error=P, table_stride=4,
                pages=8, kv_heads=2, dim=64, page_size=64, format=0, users=2, width=4, tokens=2,
                max_tokens=2, type=0)
    base.update(kw)
    return _lib.CacheCall(**base)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc required")
def test_cache_structs_match_c_layout(tmp_path):
    pairs = [("cxs_cache_call", _lib.CacheCall), ("cxs_cache_attend_call", _lib.CacheAttendCall),
             ("cxs_rotary_call", _lib.RotaryCall)]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "cxlsparse.h"',
             "int main(void) {"]
    expected = []
    for name, cls in pairs:
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            expected.append(getattr(cls, field).offset)
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        expected.append(ctypes.sizeof(cls))
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    assert [int(v) for v in out.stdout.split()] == expected


@pytest.mark.parametrize("bad,status", [
    (dict(dim=32), _lib.ERR_INVALID), (dict(page_size=128), _lib.ERR_INVALID),
    (dict(page_size=0), _lib.ERR_INVALID), (dict(format=2), _lib.ERR_INVALID),
    (dict(type=3), _lib.ERR_INVALID), (dict(pages=0), _lib.ERR_INVALID),
    (dict(kv_heads=0), _lib.ERR_INVALID), (dict(users=-1), _lib.ERR_INVALID),
    (dict(width=0), _lib.ERR_INVALID), (dict(tokens=-1), _lib.ERR_INVALID),
    (dict(max_tokens=-1), _lib.ERR_INVALID), (dict(table_stride=3), _lib.ERR_INVALID),
    (dict(offsets=None, tokens=5, max_tokens=1), _lib.ERR_INVALID),
    (dict(codes=None), _lib.ERR_INVALID), (dict(scales=None), _lib.ERR_INVALID),
    (dict(table=None), _lib.ERR_INVALID), (dict(lengths=None), _lib.ERR_INVALID),
    (dict(codes=P + 8), _lib.ERR_INVALID),
    (dict(width=1 << 25, table_stride=1 << 25), _lib.ERR_CAPACITY),
    (dict(users=70000), _lib.ERR_CAPACITY), (dict(kv_heads=40000), _lib.ERR_CAPACITY),
], ids=str)
def test_cache_calls_refuse_before_any_launch(bad, status):
    lib = _lib.lib()
    call = cache_call(**bad)
    assert lib.cxs_cache_append(call, P, 128, 64, P, 128, 64, None) == status
    assert b"cache append" in lib.cxs_last_error()
    assert lib.cxs_cache_read(call, P, P, None) == status
    heads = 2 * call.kv_heads if call.kv_heads > 0 else 4
    attend = _lib.CacheAttendCall(cache=call, query=P, out=P, q_token_stride=256,
                                  q_head_stride=64, heads=heads, scale=0.125)
    assert lib.cxs_cache_attend(attend, None) == status


def test_null_and_mismatched_arguments_are_refused():
    lib = _lib.lib()
    call = cache_call()
    assert lib.cxs_cache_append(None, P, 1, 1, P, 1, 1, None) == _lib.ERR_INVALID
    assert lib.cxs_cache_append(call, None, 1, 1, P, 1, 1, None) == _lib.ERR_INVALID
    assert lib.cxs_cache_append(call, P, 1, 1, None, 1, 1, None) == _lib.ERR_INVALID
    assert lib.cxs_cache_read(None, P, P, None) == _lib.ERR_INVALID
    assert lib.cxs_cache_read(call, P, None, None) == _lib.ERR_INVALID
    assert lib.cxs_cache_attend(None, None) == _lib.ERR_INVALID
    size = _lib.c_i64(0)
    for bad in (dict(heads=3), dict(heads=0), dict(window=-1), dict(query=None), dict(out=None)):
        fields = dict(cache=call, query=P, out=P, q_token_stride=256, q_head_stride=64, heads=4,
                      scale=0.125)
        fields.update(bad)
        assert lib.cxs_cache_attend(_lib.CacheAttendCall(**fields), None) == _lib.ERR_INVALID
    attend = _lib.CacheAttendCall(cache=cache_call(type=2), query=P, out=P, heads=4)
    assert lib.cxs_cache_attend_workspace(attend, size) == _lib.ERR_INVALID
    assert b"bf16 or fp16" in lib.cxs_last_error()
    attend = _lib.CacheAttendCall(cache=call, heads=4)
    assert lib.cxs_cache_attend_workspace(attend, size) == _lib.OK and size.value >= 0
    assert lib.cxs_cache_attend_workspace(attend, None) == _lib.ERR_INVALID
    # Nothing to do is no error, whatever the pointers.
    empty = cache_call(tokens=0, max_tokens=0, codes=None)
    assert lib.cxs_cache_append(empty, None, 0, 0, None, 0, 0, None) == _lib.OK
    assert lib.cxs_cache_read(empty, None, None, None) == _lib.OK
    assert lib.cxs_cache_attend(_lib.CacheAttendCall(cache=empty, heads=4), None) == _lib.OK


@pytest.mark.parametrize("bad", [
    dict(dim=63), dict(dim=514), dict(dim=0), dict(rotary_dim=66), dict(rotary_dim=7),
    dict(rotary_dim=0), dict(layout=2), dict(type=3), dict(tokens=-1), dict(heads=-1),
    dict(q=None), dict(k_out=None), dict(positions=None), dict(steps=None),
], ids=str)
def test_rotary_call_refusals(bad):
    fields = dict(q=P, k=P, q_out=P, k_out=P, positions=P, steps=P, tokens=2, heads=4, kv_heads=1,
                  dim=64, rotary_dim=64, layout=0, type=0, magnitude=1.0)
    fields.update(bad)
    assert _lib.lib().cxs_rotary(_lib.RotaryCall(**fields), None) == _lib.ERR_INVALID
    assert b"rotary" in _lib.lib().cxs_last_error()
    assert _lib.lib().cxs_rotary(None, None) == _lib.ERR_INVALID


def test_cache_object_refusals():
    make = lambda **kw: QuantizedCache(4, 2, 64, device="cpu", **kw)  # noqa: E731
    cache = make()
    assert cache.codes.dtype == torch.float8_e4m3fn and cache.codes.shape == (4, 2, 2, 64, 64)
    assert make(format="int8").codes.dtype == torch.int8
    for kw in (dict(format="e5m2"), dict(page_size=48)):
        with pytest.raises(ValueError):
            make(**kw)
    for args in ((0, 2, 64), (4, 0, 64), (4, 2, 96), (None, 2, 64)):
        with pytest.raises(ValueError):
            QuantizedCache(*args, device="cpu")
    codes, scales = cache.codes, cache.scales
    for c, s in ((codes, None), (codes.view(torch.uint8), scales), (codes[:, :, :1], scales),
                 (codes, scales[:3]), (codes, scales.double()), (codes[:, :, :, :40], scales),
                 (codes[..., :32], scales), (codes[:, :1], scales[:, :1])):
        with pytest.raises(ValueError):
            QuantizedCache(codes=c, scales=s)
    table = torch.zeros(2, 3, dtype=torch.int32)
    lengths, offsets = torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 2]).int()
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for args in (
            (k, k, table.long(), lengths, offsets), (k, k, table[0], lengths, offsets),
            (k, k, table, lengths[:1], offsets), (k, k, table, lengths.long(), offsets),
            (k, k, table, lengths, offsets[:2]), (k, k, table, lengths, offsets.long()),
            (k[:1], k[:1], table, lengths, None), (k, k.half(), table, lengths, offsets),
            (k, k[:1], table, lengths, offsets), (k[:, :1], k, table, lengths, offsets),
            (k[..., :32], k, table, lengths, offsets), (k.double(), k.double(), table, lengths,
                                                        offsets),
            (k.transpose(1, 2), k, table, lengths, offsets)):
        with pytest.raises(ValueError):
            cache.append(*args)
    with pytest.raises(ValueError):
        cache.append(k, k, table, lengths, offsets, max_tokens=-1)
    with pytest.raises(ValueError):
        cache.read(table, lengths, offsets, total=2, dtype=torch.float64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    for bad, kw in ((q.float(), {}), (q[:, :3], {}), (q, dict(window=-1)),
                    (q, dict(scale=math.inf)), (q[..., :32], {})):
        with pytest.raises(ValueError):
            cache.attend(bad, table, lengths, offsets, **kw)


def test_rotary_object_refusals():
    for args, kw in (((63,), {}), ((64,), dict(rotary_dim=66)), ((64,), dict(rotary_dim=7)),
                     ((64,), dict(layout="pairs")), ((64,), dict(scaling=dict(type="log"))),
                     ((64,), dict(scaling=dict(factor=2))), ((514,), {}), ((64,), dict(theta=1.0)),
                     ((64,), dict(scaling=dict(type="linear", factor=0))),
                     ((64,), dict(scaling=dict(type="linear", factor=2, original=9))),
                     ((64,), dict(scaling=dict(type="yarn", factor=2)))):
        with pytest.raises(ValueError):
            Rotary(*args, device="cpu", **kw)
    rotary = Rotary(64, device="cpu")
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 1, 64)
    p = torch.zeros(3, dtype=torch.int32)
    for args, kw in (((None, None, p), {}), ((q, k[:2], p), {}), ((q, k, p[:2]), {}),
                     ((q, k.half(), p), {}), ((q, k, p.float()), {}), ((q[..., :32], k, p), {}),
                     ((q.double(), None, p), {}), ((q.transpose(1, 2), None, p), {}),
                     ((q, k, p), dict(out=(q, None))), ((q, k, p), dict(out=(k, k)))):
        with pytest.raises(ValueError):
            rotary.apply(*args, **kw)


def test_frequencies():
    """Known values of each scaling; phases as 64-bit fractions."""
    f, m = frequencies(64)
    assert m == 1 and f[0] == 1 and math.isclose(f[16], 0.01)
    linear, m = frequencies(64, scaling=dict(type="linear", factor=4.0))
    assert m == 1 and torch.allclose(linear * 4, f)
    ntk, m = frequencies(64, scaling=dict(type="ntk", factor=8.0))
    assert m == 1 and ntk[0] == 1 and math.isclose(ntk[-1] * 8, f[-1], rel_tol=1e-12)
    yarn, m = frequencies(64, scaling=dict(type="yarn", factor=4.0, original=4096))
    assert math.isclose(m, 0.1 * math.log(4) + 1)
    turns = 4096 * f / (2 * math.pi)
    ratio = yarn / f
    assert torch.allclose(ratio[turns > 40], torch.ones(1).double())
    assert torch.allclose(ratio[turns < 0.7], torch.full((1,), 0.25).double())
    assert ((ratio[1:] <= ratio[:-1] + 1e-12)).all()
    steps = Rotary(64, device="cpu").steps
    for position in (1, 12345, 2 ** 31 - 1):
        phase = (steps * position).double() * 2.0 ** -64       # wraps, as the kernel's does
        want = f / (2 * math.pi) * position
        off = phase - want
        assert ((off - off.round()).abs() <= position * 2.0 ** -55 + 1e-9).all()
