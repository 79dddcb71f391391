"""Drawn tokens against the fp64 form: the same token, always."""

import math

import numpy
import pytest
import torch

from cxlsparse_b200.sampling import sample
from sampling_case import draw

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def same(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One call against the plain form. Log-probabilities: a sum of positive
    terms in fp32, at most (vocabulary / 32 K + 12) roundings one after another,
    an exponential of 2 units each and a logarithm: 2^-18 absolute, and two
    roundings of the value."""
    settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    tokens, logprobs = sample(logits, uniforms, return_logprobs=True, **settings)
    assert tokens.shape == uniforms.shape and tokens.dtype == torch.int64
    assert torch.equal(tokens, sample(logits, uniforms, **settings))
    rows = len(logits)
    x, u = logits.double().cpu().numpy(), uniforms.double().view(rows, -1).cpu().numpy()
    got, prob = tokens.view(rows, -1).cpu().numpy(), logprobs.view(rows, -1).cpu().double().numpy()
    for r in range(rows):
        each = {k: v[r].item() if torch.is_tensor(v) else v for k, v in settings.items()}
        want, logs = draw(x[r], u[r], **each)
        assert got[r].tolist() == want.tolist(), (r, each)
        want = numpy.where(want < 0, -numpy.inf, logs[want])
        with numpy.errstate(invalid="ignore"):
            off = numpy.where(prob[r] == want, 0.0, numpy.abs(prob[r] - want))
        assert (off <= 2.0 ** -18 + 2.0 ** -22 * numpy.abs(want)).all()
    return tokens


SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(temperature=0.6, top_k=7),
            dict(top_p=0.9), dict(top_p=0.3, temperature=2.0), dict(min_p=0.05),
            dict(top_k=50, top_p=0.95, min_p=0.01, temperature=0.8), dict(top_p=0.0),
            dict(min_p=1.0), dict(top_k=1 << 30), dict(top_k=600, top_p=0.999)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 32000])
def test_settings(cuda, vocab, settings):
    for i, dtype in enumerate(TYPES):
        g = generator(vocab + i)
        x = (3 * torch.randn(9, vocab, generator=g, device="cuda")).to(dtype)
        u = torch.rand(9, generator=g, device="cuda")
        u[0], u[1], u[2], u[3], u[4] = 0.0, 1 - 2 ** -24, 1.0, -1.0, math.nan
        same(x, u, **settings)


@pytest.mark.parametrize("rows,vocab", [(1, 131071), (3, 262145), (150, 4001), (700, 129)])
def test_rows_and_vocabularies(cuda, rows, vocab):
    """Odd sizes, rows that begin inside a 16-byte vector, many draws, fp64 numbers."""
    g = generator(rows)
    for dtype in TYPES:
        x = (2 * torch.randn(rows, vocab + 5, generator=g, device="cuda")).to(dtype)[:, 3:vocab + 3]
        u = torch.rand(rows, 3 if rows > 9 else 40, generator=g, device="cuda",
                       dtype=torch.float64)
        same(x, u, top_p=0.8)
        same(x, u)
        same(x, u[:, 0].float().contiguous(), top_k=100, min_p=0.001)


def test_every_row_its_own_settings(cuda):
    g = generator(5)
    x = (3 * torch.randn(64, 5000, generator=g, device="cuda")).to(torch.bfloat16)
    u = torch.rand(64, 5, generator=g, device="cuda")

    def pick(values, dtype):
        return torch.tensor([values[i % len(values)] for i in range(64)], dtype=dtype, device="cuda")

    tokens = same(x, u, pick([1.0, 0.0, 0.7, 1.5, -1.0, math.inf, math.nan], torch.float32),
                  pick([0, 40, 1, 4999, 5000, 5001, -3, 2, 700], torch.int32),
                  pick([1.0, 0.9, 0.5, 0.0, 2.0, math.nan, -0.1, 0.99], torch.float32),
                  pick([0.0, 0.1, 1.0, 0.001, 2.0], torch.float32))
    assert (tokens == -1).any() and (tokens >= 0).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits(cuda, dtype):
    """Ties go to the lowest index, also where thousands of equal logits stand at
    the border of a cut; zeros of both signs are equal."""
    x = torch.zeros(6, 50000, device="cuda")
    x[1, ::2] = -0.0
    x[2, 700:40000] = 1.0
    x[3, ::7] = 2.5
    x[3, 1::7] = -2.5
    x[4] = torch.arange(50000, device="cuda") % 3
    x[5, :20000] = -math.inf
    x = x.to(dtype)
    u = torch.rand(6, 9, generator=generator(1), device="cuda")
    u[:, 0], u[:, 1] = 0.0, 1.0
    for settings in (dict(top_k=3000), dict(top_p=0.37), dict(top_k=17), dict(min_p=1.0),
                     dict(top_k=20000, top_p=0.5, temperature=0.3), dict(temperature=0.0),
                     dict(top_k=6000, top_p=0.9)):
        same(x, u, **settings)


def test_near_ties_in_one_bin(cuda):
    """fp32 logits so close that one bin of the histogram holds them all, and
    logits so far apart that most have no weight."""
    g = generator(2)
    x = torch.rand(4, 60000, generator=g, device="cuda")
    x[0] = 5 + x[0] * 1e-3
    x[1] = 5 + (x[1] * 40).round() * 2.0 ** -20
    x[2] = x[2] * 1e4
    x[3] = -1e30 + x[3] * 1e25
    u = torch.rand(4, 9, generator=g, device="cuda")
    for settings in (dict(), dict(top_k=1234), dict(top_p=0.61), dict(top_k=30000, top_p=0.2),
                     dict(temperature=1e-3, top_p=0.9), dict(temperature=1e-30, top_k=5),
                     dict(temperature=1e30, top_k=900, top_p=0.5)):
        same(x, u, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_and_infinite_logits(cuda, dtype):
    g = generator(3)
    x = torch.randn(9, 3001, generator=g, device="cuda")
    x[0] = -math.inf                                    # nothing left
    x[1] = math.nan
    x[2, :3000] = -math.inf                             # one left, the last
    x[3, 5:] = -math.inf
    x[4, 100] = math.inf
    x[5, 200:203] = math.inf
    x[6, ::2] = math.nan
    x[7] = torch.finfo(dtype).min                       # a mask of the lowest value
    x[7, 77] = 1.0
    x[8] = torch.finfo(dtype).min
    x = x.to(dtype)
    u = torch.rand(9, 7, generator=g, device="cuda")
    u[:, 0], u[:, 1] = 0.0, 1.0
    for settings in SETTINGS:
        tokens = same(x, u, **settings)
        assert (tokens[:2] == -1).all() and (tokens[2] == 3000).all() and (tokens[3] < 5).all()
        assert (tokens[4] == 100).all() and (tokens[5] // 100 == 2).all()
        assert (tokens[6] % 2 == 1).all() and (tokens[7] == 77).all()


@pytest.mark.parametrize("vocab", [300, 40000])
def test_log_probability_of_a_nearly_certain_token(cuda, vocab):
    """log(1 + e) for a small e keeps its bits: e is a sum of positive terms in
    fp32 (at most 2^-18 off), whatever is 1 beside it."""
    x = torch.randn(4, vocab, generator=generator(8), device="cuda")
    for r, high in enumerate((18.0, 24.0, 30.0, 40.0)):
        x[r, 7 * r] = high
    u = torch.full((4,), 0.5, device="cuda")
    for settings in (dict(), dict(top_k=5), dict(top_p=0.9), dict(temperature=0.0)):
        tokens, logprobs = sample(x, u, return_logprobs=True, **settings)
        assert tokens.tolist() == [0, 7, 14, 21]
        far = (x.double() - x.double().amax(-1, keepdim=True)).exp()
        far[far == 1] = 0
        want = -torch.log1p(far.sum(-1))
        assert ((logprobs.double() - want).abs() <= 2.0 ** -17 * want.abs()).all()


def test_empty_calls_and_repeated_rows(cuda):
    x = torch.randn(2, 100, device="cuda")
    assert sample(x[:0], torch.rand(0, device="cuda")).shape == (0,)
    assert sample(x, torch.rand(2, 0, device="cuda")).shape == (2, 0)
    u = torch.rand(5, 2, generator=generator(4), device="cuda")
    same(x[:1].expand(5, 100), u, top_p=0.9)


def test_captured_and_on_another_stream(cuda):
    g = generator(6)
    x = (3 * torch.randn(20, 32000, generator=g, device="cuda")).to(torch.bfloat16)
    u = torch.rand(20, generator=g, device="cuda")
    settings = dict(temperature=0.7, top_k=60, top_p=0.9)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        tokens = sample(x, u, **settings)
    for _ in range(3):
        u.copy_(torch.rand(20, generator=g, device="cuda"))
        x.copy_(x.flip(0) * 0.9)
        graph.replay()
        assert torch.equal(tokens, same(x, u, **settings))
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = sample(x, u, **settings)
    stream.synchronize()
    assert torch.equal(tokens, other)
