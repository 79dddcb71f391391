"""Attention over common tokens against every user's own attention in fp64."""

import math

import pytest
import torch

from cache8_case import attend, offsets_of
from cxlsparse_b200 import CxsError
from cxlsparse_b200.quantized import QuantizedCache
from shared_case import family

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def queries(tokens, heads, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(tokens, heads, dim, generator=g, device="cuda").to(dtype)


def close(got, want, tol):
    same = (got == want) | (got.isnan() & want.isnan())
    assert (same | ((got - want).abs() <= tol)).all(), \
        ((got - want).abs() - tol).nan_to_num().max().item()


def agree(case, q, causal=True, scale=None, finite=None, **kw):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    cache = QuantizedCache(codes=case["codes"], scales=case["scales"])
    out, lse = cache.attend_shared(q, *case["call"], causal=causal, scale=scale, return_lse=True,
                                   **kw)
    cache.check()
    want, want_lse, tol, tol_lse = attend(q, case["codes"], case["scales"], case["table"],
                                          case["lengths"], case["new"], causal=causal, window=0,
                                          scale=scale)
    if finite is not None:  # tolerances of what is not NaN, from codes without NaN
        _, _, tol, tol_lse = attend(q, finite, case["scales"], case["table"], case["lengths"],
                                    case["new"], causal=causal, window=0, scale=scale)
    close(out.double(), want, tol)
    close(lse.double(), want_lse, tol_lse)
    again = cache.attend_shared(q, *case["call"], causal=causal, scale=scale, **kw)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    return out, lse


GROUPS = {
    "candidates": [(1000, [(i % 9, 1) for i in range(40)])],
    "one token of many": [(2049, [(0, 1)] * 300)],
    "edges of runs and pages": [(n, [(0, 1), (15, 1), (16, 2), (17, 30), (63, 1), (1, 64)])
                                for n in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200)],
    "nothing in common": [(0, [(5, 40), (0, 1), (300, 70)]), (0, [(100, 100)])],
    "alone": [(777, [(20, 130)]), (128, [(0, 40)])],
    "without rows": [(300, [(3, 0), (4, 50), (0, 0), (9, 60), (7, 0)]), (64, [(1, 0), (2, 0)]),
                     (50, [(1, 90), (2, 1)])],
    "long own": [(130, [(1500, 3), (7, 90), (900, 1), (0, 30)])],
}


@pytest.mark.parametrize("heads,kv_heads,dim,page_size,format,dtype", [
    (32, 2, 64, 64, "e4m3", torch.bfloat16), (8, 2, 64, 16, "int8", torch.float16),
    (16, 4, 128, 32, "e4m3", torch.float16), (8, 8, 128, 64, "int8", torch.bfloat16),
    (12, 1, 64, 32, "e4m3", torch.bfloat16)])
@pytest.mark.parametrize("name", GROUPS)
def test_groups(cuda, name, heads, kv_heads, dim, page_size, format, dtype):
    case = family(GROUPS[name], kv_heads=kv_heads, dim=dim, page_size=page_size, format=format)
    q = queries(sum(case["new"]), heads, dim, dtype)
    for causal in (True, False):
        agree(case, q, causal)


def test_new_tokens_among_the_common_ones(cuda):
    """What a row may not see is taken as its own, whatever `shared` says."""
    case = family([(200, [(0, 40)] * 9), (90, [(0, 100)] * 2)], kv_heads=2, dim=64, page_size=16,
                  format="e4m3")
    # All 240 (190) tokens of a group's users are the same.
    size, table, raw = 16, case["table"], case["codes"].view(torch.uint8)
    for low, high, common in ((0, 9, 240), (9, 11, 190)):
        for b in range(low + 1, high):
            for j in range(-(-common // size)):
                raw[table[b, j].item()] = raw[table[low, j].item()]
                case["scales"][table[b, j].item()] = case["scales"][table[low, j].item()]
    q = queries(sum(case["new"]), 16, 64, torch.bfloat16)
    call = case["call"]
    for shared in ([240, 190], [500, 500], [201, 91], [239, 1], [-3, 0]):
        case["call"] = call[:4] + (ints(shared),)
        if min(shared) >= 0:
            agree(case, q)
            agree(case, q, causal=False)
        else:
            cache = QuantizedCache(codes=case["codes"], scales=case["scales"])
            out = cache.attend_shared(q, *case["call"])
            with pytest.raises(CxsError, match="lengths or offsets"):
                cache.check()
            want = attend(q, case["codes"], case["scales"], table, case["lengths"], case["new"],
                          causal=True, window=0, scale=0.125)
            close(out.double(), want[0], want[2])


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales_strides_and_single_tokens(cuda, scale):
    case = family([(500, [(n, 1) for n in range(30)]), (77, [(n, 1) for n in range(50)])],
                  kv_heads=2, dim=128, page_size=32, format="e4m3", spread=3.0)
    wide = queries(80, 70, 131, torch.bfloat16)
    q = wide[:, 3:67, 1:129]                            # rows off 16-byte boundaries
    agree(case, q, scale=scale)
    table, lengths, offsets, groups, shared = case["call"]
    case["call"] = (table, lengths, None, groups, shared)
    agree(case, q.contiguous(), scale=scale, max_tokens=1)


def test_rows_that_see_nothing(cuda):
    """More new rows than tokens: rows before the first position get 0."""
    case = family([(20, [(0, 3), (5, 2)]), (0, [(0, 2), (0, 9)])], kv_heads=1, dim=64,
                  page_size=16, format="int8")
    table, _, _, groups, shared = case["call"]
    new = [40, 2, 10, 9]
    case["new"], case["call"] = new, (table, ints(case["lengths"]), offsets_of(new), groups, shared)
    q = queries(61, 16, 64, torch.float16)
    out, lse = agree(case, q)
    assert (out[:17] == 0).all() and (lse[:17] == -math.inf).all()
    assert (out[42:50] == 0).all() and (lse[42:50] == -math.inf).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_nan_reaches_the_rows_that_see_it(cuda, dim):
    """NaN codes of V among the common tokens, and among some users' own."""
    case = family([(300, [(n, 2) for n in range(40)])], kv_heads=2, dim=dim, page_size=32,
                  format="e4m3")
    finite = case["codes"].clone()
    raw, table = case["codes"].view(torch.uint8), case["table"]
    raw[table[0, 2].item(), 0, 1, 5, 7] = 0x7F           # token 69: all rows
    raw[table[9, 9].item(), 1, 1, 300 % 32 + 3, 11] = 0xFF   # token 303: user 9's rows
    q = queries(80, 32, dim, torch.bfloat16)
    out, lse = agree(case, q, finite=finite)
    assert out[:, :16, 7].isnan().all() and not out[:, :16, 8].isnan().any()
    assert out[18:20, 16:, 11].isnan().all()
    assert not out[:18, 16:].isnan().any() and not out[20:, 16:].isnan().any()
    assert lse.isfinite().all()


@pytest.mark.parametrize("kv_heads,dim,format", [(2, 64, "e4m3"), (8, 128, "int8"),
                                                 (2, 128, "e4m3")])
def test_scales_that_are_no_numbers_stay_with_their_user(cuda, kv_heads, dim, format):
    """Own pages whose scales are NaN or infinite: no other user's row sees them."""
    case = family([(256, [(20 + n, 1) for n in range(40)])], kv_heads=kv_heads, dim=dim,
                  page_size=32, format=format)
    q = queries(40, 16, dim, torch.bfloat16)
    want, want_lse, tol, tol_lse = attend(q, case["codes"], case["scales"], case["table"],
                                          case["lengths"], case["new"], causal=True, window=0,
                                          scale=0.1)
    for user, value in ((3, math.nan), (17, math.inf), (18, -math.inf), (39, math.nan)):
        for page in case["table"][user, 8:].tolist():
            if page >= 0:
                case["scales"][page] = value
    cache = QuantizedCache(codes=case["codes"], scales=case["scales"])
    out, lse = cache.attend_shared(q, *case["call"], scale=0.1, return_lse=True)
    cache.check()
    others = [n for n in range(40) if n not in (3, 17, 18, 39)]
    close(out[others].double(), want[others], tol[others])
    close(lse[others].double(), want_lse[others], tol_lse[others])
    assert not lse[[3, 17, 39]].isfinite().any()


def test_groups_that_do_not_fit(cuda):
    case = family([(100, [(n, 3) for n in range(9)]), (50, [(4, 8), (2, 30)]),
                   (80, [(1, 2)] * 12)], kv_heads=2, dim=64, page_size=16, format="e4m3")
    q = queries(sum(case["new"]), 32, 64, torch.bfloat16)
    table, lengths, offsets, groups, shared = case["call"]
    cache = QuantizedCache(codes=case["codes"], scales=case["scales"])
    want, want_lse, tol, tol_lse = attend(q, case["codes"], case["scales"], case["table"],
                                          case["lengths"], case["new"], causal=True, window=0,
                                          scale=0.125)

    def right(out, lse, rows):
        close(out[rows].double(), want[rows], tol[rows])
        close(lse[rows].double(), want_lse[rows], tol_lse[rows])

    def run(*call, **kw):
        out, lse = cache.attend_shared(q, *call, return_lse=True, **kw)
        with pytest.raises(CxsError, match="lengths or offsets"):
            cache.check()
        return out, lse

    def none(out, lse, rows):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()

    # A group with a user of more than max_tokens rows has none.
    out, lse = run(*case["call"], max_tokens=8)
    none(out, lse, slice(27, 65))
    right(out, lse, slice(0, 27))
    right(out, lse, slice(65, None))
    # Groups or offsets that do not ascend: no rows at all.
    for bad in (ints([0, 11, 9, 23]), ints([0, 9, 11, 24]), ints([-1, 9, 11, 23])):
        none(*run(table, lengths, offsets, bad, shared), slice(0, None))
    for at, value in ((3, 0), (23, 500), (0, -1)):
        wrong = offsets.clone()
        wrong[at] = value
        none(*run(table, lengths, wrong, groups, shared), slice(0, None))
    # Users of no group, rows of no user: nothing of theirs.
    out, lse = cache.attend_shared(q, table, lengths, offsets, groups + ints([9, 2, 0, 0]),
                                   shared, return_lse=True)
    none(out, lse, slice(0, 27))
    right(out, lse, slice(65, None))
    # Lengths past the table are cut to it.
    longer = lengths.clone()
    longer[0] = 10000
    out, lse = run(table, longer, offsets, groups, shared)
    right(out, lse, slice(27, None))


@pytest.mark.parametrize("gone", [[0], [0, 1, 2, 41, 79], list(range(39))])
def test_users_that_have_ended(cuda, gone):
    """Users without rows may hold nothing at all, the first of a group too."""
    case = family([(200, [(n % 7, 2) for n in range(40)])] * 2, kv_heads=2, dim=64, page_size=32,
                  format="int8")
    for user in gone:
        case["table"][user] = -1
        case["lengths"][user] = case["new"][user] = 0
    table, _, _, groups, shared = case["call"]
    case["call"] = (table, ints(case["lengths"]), offsets_of(case["new"]), groups, shared)
    agree(case, queries(sum(case["new"]), 32, 64, torch.bfloat16))


def test_bad_pages_are_left_out(cuda):
    case = family([(200, [(20, 1)] * 70)], kv_heads=1, dim=64, page_size=16, format="e4m3")
    q = queries(70, 4, 64, torch.bfloat16)
    cache = QuantizedCache(codes=case["codes"], scales=case["scales"])
    want = cache.attend_shared(q, *case["call"])
    table = case["table"].clone()
    table[3, 13] = -1                                   # own tokens 208 ..
    case["call"] = (table,) + case["call"][1:]
    out = cache.attend_shared(q, *case["call"])
    with pytest.raises(CxsError, match="page id"):
        cache.check()
    assert torch.equal(out[:3], want[:3]) and torch.equal(out[4:], want[4:])
    assert not torch.equal(out[3], want[3]) and out.isfinite().all()
    table[0, 5] = 10 ** 6                               # common tokens: of all
    out = cache.attend_shared(q, *case["call"])
    with pytest.raises(CxsError, match="page id"):
        cache.check()
    assert out.isfinite().all() and not (out == want).all(-1).all(-1).any()


def test_many_groups_and_users(cuda):
    """More groups than warps and users than threads, over few and many shares."""
    groups = [(17 * g % 230, [(i * g % 40, 1 + i % 3) for i in range(1 + g % 50)])
              for g in range(90)]
    case = family(groups, kv_heads=2, dim=64, page_size=32, format="e4m3")
    assert len(case["new"]) > 2048
    agree(case, queries(sum(case["new"]), 32, 64, torch.bfloat16))


def test_captured_with_other_lengths(cuda):
    """One captured call serves other lengths, groups and common tokens; two
    captured graphs, each with scratch of its own, run side by side."""
    first = family([(1000, [(n, 2) for n in range(40)])], kv_heads=2, dim=64, page_size=64,
                   format="e4m3")
    q = queries(80, 32, 64, torch.bfloat16)
    cache = QuantizedCache(codes=first["codes"], scales=first["scales"])
    call = tuple(t.clone() for t in first["call"])
    cache.attend_shared(q, *call)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], []
    for _ in range(2):
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(cache.attend_shared(q, *call, max_tokens=2))
        graphs.append(graph)
        streams.append(stream)
    for lengths, shared in ((first["lengths"], 1000), ([n - 30 for n in first["lengths"]], 940),
                            ([n - 1000 + 64 for n in first["lengths"]], 64)):
        call[1].copy_(ints(lengths))
        call[4].copy_(ints([shared]))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want, _, tol, _ = attend(q, first["codes"], first["scales"], first["table"], lengths,
                                 first["new"], causal=True, window=0, scale=0.125)
        for out in outs:
            close(out.double(), want, tol)
    cache.check()


def test_little_to_do(cuda):
    cache = QuantizedCache(4, 2, 64)
    empty = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    none = ints([])
    out = cache.attend_shared(empty, ints([]).view(0, 1), none, ints([0]), ints([0]), none)
    assert out.shape == (0, 4, 64)
    out = cache.attend_shared(empty, ints([[0], [1]]), ints([1, 1]), ints([0, 0, 0]), ints([0, 2]),
                              ints([1]))
    assert out.shape == (0, 4, 64)
