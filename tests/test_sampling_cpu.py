"""Refusals of the sampling call, without a device."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cxlsparse_b200 import _lib
from cxlsparse_b200.sampling import sample

HEADER = Path(__file__).resolve().parent.parent / "include" / "cxlsparse.h"
P = 4096  # an address that is never followed


def sample_call(**kw):
    base = dict(logits=P, uniforms=P, tokens=P, logprobs=P, row_stride=100, rows=2, vocab=100,
                draws=1, type=0, temperature_all=1.0, top_p_all=1.0)
    base.update(kw)
    return _lib.SampleCall(**base)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc required")
def test_sample_struct_matches_c_layout(tmp_path):
    fields = [name for name, _ in _lib.SampleCall._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "cxlsparse.h"',
             "int main(void) {"]
    lines += [f'printf("%zu\\n", offsetof(cxs_sample_call, {f}));' for f in fields]
    lines += ['printf("%zu\\n", sizeof(cxs_sample_call));', "return 0; }"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    want = [getattr(_lib.SampleCall, f).offset for f in fields] + [ctypes.sizeof(_lib.SampleCall)]
    assert [int(v) for v in out.stdout.split()] == want


@pytest.mark.parametrize("bad,status", [
    (dict(rows=-1), _lib.ERR_INVALID), (dict(vocab=0), _lib.ERR_INVALID),
    (dict(draws=-1), _lib.ERR_INVALID), (dict(type=3), _lib.ERR_INVALID),
    (dict(vocab=(1 << 24) + 1), _lib.ERR_CAPACITY),
    (dict(rows=1 << 24, draws=1 << 8), _lib.ERR_CAPACITY),
    (dict(temperature_all=-1.0), _lib.ERR_INVALID),
    (dict(temperature_all=math.nan), _lib.ERR_INVALID),
    (dict(temperature_all=math.inf), _lib.ERR_INVALID), (dict(top_k_all=-1), _lib.ERR_INVALID),
    (dict(top_p_all=-0.5), _lib.ERR_INVALID), (dict(top_p_all=math.nan), _lib.ERR_INVALID),
    (dict(min_p_all=1.5), _lib.ERR_INVALID), (dict(min_p_all=-0.5), _lib.ERR_INVALID),
    (dict(logits=None), _lib.ERR_INVALID), (dict(uniforms=None), _lib.ERR_INVALID),
    (dict(tokens=None), _lib.ERR_INVALID), (dict(logits=P + 1), _lib.ERR_INVALID),
    (dict(logits=P + 2, type=2), _lib.ERR_INVALID),
], ids=str)
def test_sample_refuses_before_any_launch(bad, status):
    lib = _lib.lib()
    assert lib.cxs_sample(sample_call(**bad), None) == status
    assert b"sample" in lib.cxs_last_error()


def test_nothing_to_draw_is_no_error():
    lib = _lib.lib()
    assert lib.cxs_sample(None, None) == _lib.ERR_INVALID
    assert lib.cxs_sample(sample_call(rows=0, logits=None), None) == _lib.OK
    assert lib.cxs_sample(sample_call(draws=0, tokens=None), None) == _lib.OK


def test_sample_arguments():
    x, u = torch.zeros(3, 8), torch.zeros(3)
    ints, floats = torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    for args, kw in (
            ((x[0], u), {}), ((x.double(), u), {}), ((x.t(), torch.zeros(8)), {}),
            ((x[:, :0], u), {}), ((x, u[:2]), {}), ((x, u.half()), {}),
            ((x, torch.zeros(3, 2, 1)), {}), ((x, torch.zeros(3, 4)[:, ::2]), {}),
            ((x.requires_grad_(), u), {}), ((x, u), dict(temperature=-1)),
            ((x, u), dict(temperature=math.inf)), ((x, u), dict(temperature=math.nan)),
            ((x, u), dict(top_k=-1)), ((x, u), dict(top_p=-0.1)), ((x, u), dict(top_p=math.nan)),
            ((x, u), dict(min_p=1.1)), ((x, u), dict(temperature=floats.double())),
            ((x, u), dict(temperature=floats[:2])), ((x, u), dict(top_k=floats)),
            ((x, u), dict(top_p=ints)), ((x, u), dict(min_p=torch.zeros(6)[::2]))):
        with pytest.raises(ValueError):
            sample(*args, **kw)
        x = x.detach()
