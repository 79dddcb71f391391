"""Rotary positions on the device against the formula in fp64."""

import math

import pytest
import torch

from cxlsparse_b200.rotary import Rotary, frequencies

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SCALINGS = [None, dict(type="linear", factor=4.0), dict(type="ntk", factor=8.0),
            dict(type="yarn", factor=4.0, original=4096)]


def formula(x, positions, f, magnitude, layout, transpose=False):
    """(rotated x, sum of magnitudes behind each element) in fp64."""
    x, d = x.double(), 2 * len(f)
    angle = positions.double()[:, None, None] * f.to(x.device)
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude
    if transpose:
        sin = -sin
    if layout == "half":
        a, b = x[..., :d // 2], x[..., d // 2:d]
        join = lambda u, w: torch.cat((u, w), -1)  # noqa: E731
    else:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
        join = lambda u, w: torch.stack((u, w), -1).flatten(-2)  # noqa: E731
    size = (a.abs() + b.abs()) * magnitude
    turned = join(a * cos - b * sin, b * cos + a * sin)
    rest = x[..., d:]
    return torch.cat((turned, rest), -1), torch.cat((join(size, size), 0 * rest), -1)


def close(got, want, size, dtype):
    """Phases are rounded to 24 bits of a half turn (pi 2^-24), sine and cosine
    are within 2 units of 2^-23, the two products and the sum within 2^-23
    together: 6e-7 of |a| + |b|; then one rounding to the type."""
    off = (got.double() - want).abs()
    assert (off <= UNIT[dtype] * want.abs() + 6e-7 * size + 1e-30
            + (2.0 ** -25 if dtype == torch.float16 else 0.0)).all(), off.max()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (128, 128), (128, 64), (64, 48), (128, 112),
                                            (80, 20), (6, 2), (512, 512), (130, 66)])
@pytest.mark.parametrize("tokens", [1, 3, 65])
def test_rotary_matches_formula(cuda, layout, dtype, dim, rotary_dim, tokens):
    g = torch.Generator(device="cuda").manual_seed(dim + tokens)
    q = torch.randn(tokens, 5, dim, generator=g, device="cuda").to(dtype)
    k = torch.randn(tokens, 2, dim, generator=g, device="cuda").to(dtype)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    positions[0] = 0
    positions[-1] = 131071
    for scaling in SCALINGS:
        for transpose in (False, True):
            rotary = Rotary(dim, rotary_dim=rotary_dim, layout=layout, scaling=scaling)
            f, magnitude = frequencies(rotary_dim, scaling=scaling)
            for p in (positions, positions.int()):
                got = rotary.apply(q, k, p, transpose=transpose)
                for x, y in zip((q, k), got):
                    want, size = formula(x, positions, f, magnitude, layout, transpose)
                    close(y, want, size, dtype)
                    assert torch.equal(y[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_holds_at_long_positions(cuda, layout):
    """Positions near 2^31 and below zero keep full fp32 accuracy."""
    positions = torch.tensor([0, 1, -1, 2 ** 20 + 1, 2 ** 31 - 1, -2 ** 31], device="cuda")
    q = torch.randn(6, 4, 64, device="cuda")
    f, magnitude = frequencies(64)
    got, _ = Rotary(64, layout=layout).apply(q, None, positions)
    want, size = formula(q, positions, f, magnitude, layout)
    # fp64 angles of 2^31 radians are off by 2^31 * 2^-53 themselves.
    assert ((got.double() - want).abs() <= 6e-7 * size + 2.0 ** -24 * want.abs() + 1e-6).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_strides_in_place_and_one_tensor(cuda, layout, dtype):
    tokens, heads, kv, dim = 37, 6, 2, 64
    proj = torch.randn(tokens, (heads + 2 * kv) * dim + 3, device="cuda").to(dtype)
    positions = torch.arange(5000, 5000 + tokens, device="cuda", dtype=torch.int32)
    rotary = Rotary(dim, layout=layout)
    for shift in (0, 1):                     # 16-byte aligned, then not
        rows = proj[:, shift:]
        q = rows[:, :heads * dim].view(tokens, heads, dim)
        k = rows[:, heads * dim:(heads + kv) * dim].view(tokens, kv, dim)
        want = rotary.apply(q.contiguous(), k.contiguous(), positions)
        assert all(torch.equal(x, y) for x, y in zip(rotary.apply(q, k, positions), want))
        alone_q, none = rotary.apply(q, None, positions)
        none_q, alone_k = rotary.apply(None, k, positions)
        assert none is None and none_q is None
        assert torch.equal(alone_q, want[0]) and torch.equal(alone_k, want[1])
        swapped = q.transpose(0, 1).contiguous().transpose(0, 1)       # heads outermost
        assert torch.equal(rotary.apply(swapped, None, positions)[0], want[0])
        spaced = torch.empty(2 * tokens, dtype=torch.int32, device="cuda")[::2]
        spaced.copy_(positions)
        assert torch.equal(rotary.apply(q, None, spaced)[0], want[0])
        copy = proj.clone()[:, shift:]
        q2 = copy[:, :heads * dim].view(tokens, heads, dim)
        k2 = copy[:, heads * dim:(heads + kv) * dim].view(tokens, kv, dim)
        out = rotary.apply(q2, k2, positions, out=(q2, k2))
        assert out[0] is q2 and torch.equal(q2, want[0]) and torch.equal(k2, want[1])
        assert torch.equal(copy[:, (heads + kv) * dim:], rows[:, (heads + kv) * dim:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_transposed_rotation_is_the_gradient(cuda, layout):
    """<g, R(x + e d) - R(x - e d)> / 2 e = <R^T g, d>: R is linear, so central
    differences are exact but for fp32 rounding."""
    scaling = dict(type="yarn", factor=4.0, original=4096)
    rotary = Rotary(64, rotary_dim=48, layout=layout, scaling=scaling)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, d, g = (torch.randn(33, 4, 64, generator=gen, device="cuda") for _ in range(3))
    positions = torch.randint(0, 100000, (33,), generator=gen, device="cuda")
    back, _ = rotary.apply(g, None, positions, transpose=True)
    plus, _ = rotary.apply(x + d, None, positions)
    minus, _ = rotary.apply(x - d, None, positions)
    change = (g.double() * (plus.double() - minus.double())).sum() / 2
    slope = (back.double() * d.double()).sum()
    # 8448 products of unit size, each within about 1e-6: well below 1e-2 together.
    assert abs(change - slope) <= 1e-2
    # For magnitude 1 the transposed rotation undoes the rotation.
    plain = Rotary(64, layout=layout)
    there, _ = plain.apply(x, None, positions)
    again, _ = plain.apply(there, None, positions, transpose=True)
    assert (again - x).abs().max() <= 6e-6


def test_rotary_agrees_with_the_glue_kernel(cuda):
    """The half layout over whole heads is what the extend model's glue applies
    (which rounds sine, cosine and both products to bf16)."""
    from cxlsparse_b200.model import rotary as plain

    q = torch.randn(40, 32, 64, device="cuda").bfloat16()
    k = torch.randn(40, 2, 64, device="cuda").bfloat16()
    positions = torch.arange(1000, 1040, device="cuda")
    f = (10000.0 ** (-torch.arange(0, 64, 2, device="cuda").float() / 64))
    want = plain(q, k, positions, f)
    got = Rotary(64).apply(q, k, positions)
    for x, y in zip(got, want):
        # Four bf16 roundings of values up to |a| + |b| (below 12 here).
        assert (x.float() - y.float()).abs().max() <= 4 * 2.0 ** -8 * 12


def test_no_tokens(cuda):
    q, k = Rotary(64).apply(torch.empty(0, 2, 64, device="cuda"),
                            torch.empty(0, 1, 64, device="cuda"),
                            torch.empty(0, dtype=torch.int32, device="cuda"))
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    assert math.isclose(Rotary(64, scaling=SCALINGS[3]).magnitude, 0.1 * math.log(4) + 1)
