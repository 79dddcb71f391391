"""Candidates of users' histories: pages, attention over common tokens and
sampling run together, against the same steps taken user by user."""

import pytest
import torch

from cxlsparse_b200.dense import DenseCacheModel
from cxlsparse_b200.model import NSAConfig
from cxlsparse_b200.pages import PageTable
from cxlsparse_b200.quantized import QuantizedCache
from cxlsparse_b200.sampling import sample
from shared_case import family

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=256, q_heads=8, kv_heads=2, ffn=512, vocab=500)
SETTINGS = dict(temperature=0.9, top_k=100, top_p=0.95, min_p=0.001)


def made(users, **kw):
    return DenseCacheModel(NSAConfig(**CFG), users=users, max_tokens=400, **kw)


def prompt(lengths, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 500, (sum(lengths),), generator=g, device="cuda")


def last_rows(lengths):
    return torch.tensor(lengths, device="cuda").cumsum(0) - 1


@pytest.mark.parametrize("format,page_size,lengths", [
    ("e4m3", 64, [331, 64, 7]), ("int8", 16, [16, 250]), ("e4m3", 32, [129])])
def test_candidates_follow_steps_of_users_of_their_own(cuda, format, page_size, lengths):
    """The same tokens are forced on a model in which every candidate is a user
    with the whole history, and each has to be where u falls in that model's
    distribution. The cached codes are the same; attention rounds in another
    order, so that logits (below 2 in magnitude) differ by a few roundings to
    bf16, 2^-9 each of the hidden state and of themselves: at most 0.02, and sums
    of probabilities, at temperature 1, by twice that."""
    users, count, steps = len(lengths), 12, 20
    model = made(users, page_size=page_size, format=format, candidates=16, candidate_tokens=steps)
    tokens = prompt(lengths)
    logits = model.step(tokens, lengths)[last_rows(lengths)]
    u = torch.rand(users, count, steps, generator=torch.Generator(device="cuda").manual_seed(1),
                   device="cuda")
    drawn, logprobs = model.generate(logits, u)
    model.check()
    assert drawn.shape == logprobs.shape == (users, count, steps) and drawn.dtype == torch.int64
    assert torch.equal(drawn, model.generate(logits, u)[0])

    parts = tokens.split(lengths)
    many = made(users * count, page_size=page_size, format=format)
    theirs = [n for n in lengths for _ in range(count)]
    other = many.step(torch.cat([p for p in parts for _ in range(count)]), theirs)[last_rows(theirs)]
    for step in range(steps):
        forced = drawn[:, :, step].reshape(-1, 1)
        logs = other.double().log_softmax(-1)
        upto = logs.exp().cumsum(-1).gather(1, forced)
        at = u[:, :, step].double().reshape(-1, 1)
        assert (at <= upto + 0.04).all()
        assert (at >= upto - logs.gather(1, forced).exp() - 0.04).all()
        off = logs.gather(1, forced) - logprobs[:, :, step].reshape(-1, 1)
        assert (off.abs() <= 0.04).all()
        if step + 1 < steps:
            other = many.step(forced[:, 0], [1] * len(theirs))
    cut, _ = model.generate(logits, u, **SETTINGS)
    first = sample(logits, u[:, :, 0].contiguous(), **SETTINGS)
    assert torch.equal(cut[:, :, 0], first) and (cut >= 0).all()
    # The histories are as they were: the next step does not see the candidates.
    plain = made(users, page_size=page_size, format=format)
    plain.step(tokens, lengths)
    for _ in range(2):
        got, want = (m.step(tokens[:users], [1] * users) for m in (model, plain))
        assert torch.equal(got, want)


def test_candidates_of_one_history_differ_and_repeat(cuda):
    model = made(1, candidates=64, candidate_tokens=8)
    tokens = prompt([200])
    logits = model.step(tokens, [200])[-1:]
    u = torch.rand(1, 64, 8, device="cuda")
    drawn, _ = model.generate(logits, u)
    assert len({tuple(x) for x in drawn[0].tolist()}) > 60
    greedy, _ = model.generate(logits, u, temperature=0.0)
    assert (greedy == greedy[:, :1]).all()
    assert greedy[0, 0, 0] == logits.argmax()
    model.check()


def test_settings_of_each_user(cuda):
    lengths = [70, 30, 100]
    model = made(3, candidates=4, candidate_tokens=6)
    logits = model.step(prompt(lengths), lengths)[last_rows(lengths)]
    u = torch.rand(3, 4, 6, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    heat = torch.tensor([0.0, 1.0, 0.5], device="cuda")
    most = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    tokens, _ = model.generate(logits, u, temperature=heat, top_k=most)
    for n in range(3):
        one, _ = model.generate(logits, u, temperature=heat[n].item(), top_k=most[n].item())
        assert torch.equal(tokens[n], one[n])
    assert (tokens[:2] == tokens[:2, :1]).all()
    model.check()


def test_generate_refuses(cuda):
    model = made(2, candidates=4, candidate_tokens=5)
    logits = model.step(prompt([9, 9]), [9, 9])[[8, 17]]
    u = torch.rand(2, 4, 5, device="cuda")
    for args in ((logits[:1], u), (logits, u[:1]), (logits, u[:, :0]), (logits, u[..., :0]),
                 (logits, torch.rand(2, 5, 5, device="cuda")), (logits, u[0]),
                 (logits, torch.rand(2, 4, 6, device="cuda"))):
        with pytest.raises(ValueError):
            model.generate(*args)
    with pytest.raises(ValueError):
        made(2).generate(logits, u)


def test_pages_behind_four_gigabytes(cuda):
    """The same cache at the end of a pool of 2^32 bytes: forked, attended to,
    compacted and attended to again, with results equal to the bit."""
    case = family([(300, [(n, 2) for n in range(36)])], kv_heads=8, dim=64, page_size=64,
                  format="e4m3")
    table, lengths, offsets, groups, shared = case["call"]
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(72, 64, 64, generator=g, device="cuda").bfloat16()
    small = QuantizedCache(codes=case["codes"], scales=case["scales"])
    want = small.attend_shared(q, *case["call"])
    pages, count = 66000, case["codes"].shape[0]
    large = QuantizedCache(pages, 8, 64, page_size=64, format="e4m3")
    assert large.codes.numel() > 2 ** 32
    at = pages - count
    large.codes.view(torch.uint8)[at:] = case["codes"].view(torch.uint8)
    large.scales[at:] = case["scales"]
    pool = PageTable([large], 37, table.shape[1])
    rows = torch.full((37, table.shape[1]), -1, dtype=torch.int32, device="cuda")
    rows[:36] = torch.where(table >= 0, table + at, table)
    pool.adopt(rows, torch.cat((lengths, lengths.new_zeros(1))))
    pool.fork(lengths.new_tensor([35]), lengths.new_tensor([36]))

    def agree():
        for last in (35, 36):
            order = list(range(35)) + [last]
            got = large.attend_shared(q, pool.table[order], pool.lengths[order], offsets, groups,
                                      shared)
            assert torch.equal(got, want)
        large.check()
        pool.check()

    agree()
    live = pool.compact().item()
    assert live < count + 2 and pool.table.max().item() == live - 1
    agree()


def test_rows_behind_four_gigabytes(cuda):
    vocab, stride = 50000, 2 ** 30 + 24
    g = torch.Generator(device="cuda").manual_seed(4)
    few = torch.randn(3, vocab, generator=g, device="cuda").bfloat16()
    far = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    far = far.as_strided((3, vocab), (stride, 1))
    far.copy_(few)
    u = torch.rand(3, 40, generator=g, device="cuda")
    for settings in ({}, SETTINGS, dict(top_p=0.5), dict(temperature=0.0)):
        for got, want in zip(sample(far, u, return_logprobs=True, **settings),
                             sample(few, u, return_logprobs=True, **settings)):
            assert torch.equal(got, want)
