"""Paged decode attention of values that are not finite: what a sequence attends to shows in its
output as the 64-bit formula has it, whatever the length, the cut of the work and the tile, and
in no other sequence's or head's."""

import pytest
import torch

from tests import op_reference as ref
from tests.test_gpu_operators import DEV, gen, make_cache, randn

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def put(pages, cache, i, pos, head, value, dim=None, shared=0):
    """One row of sequence i (of the shared part: of the first sequence's table row)."""
    page = cache.page_size
    at = cache.block_table[0 if pos < shared else i, pos // page].item()
    row = pages[at, head, pos % page]
    row[slice(None) if dim is None else dim] = value


def check(cache, q, clean, shared=0):
    """attend against the formula: where that is finite within the bound of `clean` (the values
    (out, bound) before something was put in; what differs has to be non-finite), elsewhere the
    same infinity or NaN."""
    got = cache.attend(q, shared_len=shared)
    cache.check_status()
    want, _ = ref.attend(q, cache.k_pages, cache.v_pages, cache.block_table, cache.lens, q.shape[-1] ** -0.5, shared)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places than the formula's"
    inf = torch.isinf(want)
    assert torch.equal(got[inf].double(), want[inf])
    over = (got.double() - clean[0]).abs() - clean[1]
    assert bool((over[finite] <= 0).all())
    return want


def formula(cache, q, shared=0):
    return ref.attend(q, cache.k_pages, cache.v_pages, cache.block_table, cache.lens, q.shape[-1] ** -0.5, shared)


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 64, 65, 128, 129, 257, 1000, 20000])
def test_a_nan_key_at_the_last_row(length):
    g = gen(length)
    cache = make_cache(g, [length, 77], 2, 64, 64)
    q = randn(g, 2, 4, 1, 64)
    clean = formula(cache, q)
    put(cache.k_pages, cache, 0, length - 1, 1, NAN, dim=9)
    want = check(cache, q, clean)
    assert torch.isnan(want[0, 0, 2:]).all() and torch.isfinite(want[0, 0, :2]).all()


@pytest.mark.parametrize("first,last", [(0, 32), (32, 64), (96, 128), (128, 160), (0, 128), (0, 300)])
def test_runs_of_nan_keys(first, last):
    g = gen(first + last)
    cache = make_cache(g, [300, 200], 1, 16, 128)
    q = randn(g, 2, 8, 1, 128)
    clean = formula(cache, q)
    for pos in range(first, last):
        put(cache.k_pages, cache, 0, pos, 0, NAN)
    assert torch.isnan(check(cache, q, clean)[0]).all()


@pytest.mark.parametrize("batch,hq,hkv,d,shared", [(3, 4, 2, 128, 0), (2, 8, 2, 64, 256), (33, 8, 2, 128, 256),
                                                   (33, 8, 8, 64, 1024), (70, 8, 1, 64, 640), (1, 1, 1, 64, 128)],
                         ids=["own", "narrow prefix", "wide prefix", "one row a sequence", "pair of tiles", "lone row"])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_a_query_that_is_not_finite(batch, hq, hkv, d, shared, value):
    g = gen(batch + d)
    cache = make_cache(g, [shared + (i * 37) % 300 + (shared == 0) for i in range(batch)], hkv, 64, d, shared=shared)
    q = randn(g, batch, hq, 1, d)
    clean = formula(cache, q, shared)
    q[batch // 2, hq - 1, 0, 3] = value
    want = check(cache, q, clean, shared)
    assert torch.isnan(want[batch // 2, 0, hq - 1]).all()


@pytest.mark.parametrize("batch", [2, 33, 70])
def test_nan_keys_of_a_shared_prefix(batch):
    """A whole chunk of the prefix NaN in one head; a sequence that ends before it is not touched."""
    g = gen(batch)
    lens = [640 + i % 50 for i in range(batch)]
    lens[1] = 100
    cache = make_cache(g, [max(n, 640) for n in lens], 2, 64, 64, shared=640)
    cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    q = randn(g, batch, 8, 1, 64)
    clean = formula(cache, q, 640)
    for pos in range(256, 384):
        put(cache.k_pages, cache, 0, pos, 1, NAN, shared=640)
    want = check(cache, q, clean, 640)
    assert torch.isnan(want[0, 0, 4:]).all() and torch.isfinite(want[1]).all()


def test_a_nan_query_of_an_idle_sequence():
    g = gen(3)
    cache = make_cache(g, [0, 200], 2, 64, 64)
    q = randn(g, 2, 4, 1, 64)
    clean = formula(cache, q)
    q[0] = NAN
    want = check(cache, q, clean)
    assert not want[0].any()


@pytest.mark.parametrize("batch,hq,hkv,d,shared", [(3, 4, 2, 128, 0), (3, 6, 2, 64, 0), (2, 8, 2, 64, 256),
                                                   (33, 8, 2, 128, 256), (70, 8, 1, 64, 640)],
                         ids=["own", "own of odd groups", "narrow prefix", "wide prefix", "pair of tiles"])
@pytest.mark.parametrize("values", [(INF,), (-INF,), (INF, INF), (INF, -INF), (NAN, INF), (NAN,)],
                         ids=["inf", "-inf", "two", "both signs", "with nan", "nan"])
def test_values_that_are_not_finite(batch, hq, hkv, d, shared, values):
    """An infinite value gives an infinite output in its dim, NaN only beside a NaN or one of the
    other sign; once in the first rows, once in the last."""
    g = gen(batch + d)
    lens = [shared + 200 + (i * 37) % 300 for i in range(batch)]
    cache = make_cache(g, lens, hkv, 64, d, shared=shared)
    q = randn(g, batch, hq, 1, d)
    clean = formula(cache, q, shared)
    for n, value in enumerate(values):
        put(cache.v_pages, cache, 1, 40 + 50 * n, hkv - 1, value, dim=7, shared=shared)
        put(cache.v_pages, cache, 1, lens[1] - 1 - 33 * n, 0, value, dim=d - 1)
    want = check(cache, q, clean, shared)
    assert not torch.isfinite(want[1, 0, -1, 7]) and not torch.isfinite(want[1, 0, 0, d - 1])


@pytest.mark.parametrize("shared", [0, 128])
def test_an_infinite_value_of_small_probability(shared):
    """A probability that its 16-bit type rounds to 0 still gives its infinity: scores about 30
    below the largest, 2^-43."""
    g = gen(5)
    cache = make_cache(g, [200, 150], 1, 32, 64, torch.float16, shared=shared)
    q = randn(g, 2, 2, 1, 64, dtype=torch.float16)
    put(cache.k_pages, cache, 0, 70, 0, (q[0, 0, 0] * 240 / q[0, 0, 0].square().sum()), shared=shared)
    put(cache.k_pages, cache, 0, 71, 0, 0.0, shared=shared)
    clean = formula(cache, q, shared)
    put(cache.v_pages, cache, 0, 71, 0, -INF, dim=11, shared=shared)
    assert check(cache, q, clean, shared)[0, 0, 0, 11] == -INF


@pytest.mark.parametrize("batch,shared,own", [(2, 0, 1), (2, 0, 130), (2, 0, 1000), (2, 128, 40), (33, 256, 20)])
def test_scores_that_are_all_minus_infinity(batch, shared, own):
    """A softmax over nothing but -infinity is 0 / 0, NaN; some of them alone are left out."""
    g = gen(batch + own)
    cache = make_cache(g, [shared + own + i for i in range(batch)], 2, 64, 128, shared=shared)
    q = randn(g, batch, 4, 1, 128)
    q[0, 2:, 0, 3] = 1.0
    for pos in range(shared + own):
        put(cache.k_pages, cache, 0, pos, 1, -INF, dim=3, shared=shared)
    want, _ = formula(cache, q, shared)
    got = cache.attend(q, shared_len=shared)
    assert torch.isnan(got[0, 0, 2:]).all() and torch.isnan(want[0, 0, 2:]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(want))


def test_some_scores_of_minus_infinity_count_as_nothing():
    """Bound: that of the formula over the rows that are left."""
    g = gen(9)
    lens, out = [300, 200], (0, 1, 2, 5, 140, *range(160, 192), 299)
    cache = make_cache(g, lens, 2, 64, 128)
    q = randn(g, 2, 4, 1, 128)
    q[0, 2:, 0, 3] = 1.0
    left = make_cache(gen(10), [300 - len(out)], 2, 64, 128)
    for pages, to in ((cache.k_pages, left.k_pages), (cache.v_pages, left.v_pages)):
        rows = ref.gather(pages, cache.block_table[0], 300)
        rows = rows[:, [p for p in range(300) if p not in out]]
        for n in range(rows.shape[1]):
            to[int(left.block_table[0, n // 64]), :, n % 64] = rows[:, n].to(to.dtype)
    want, bound = formula(left, q[:1])
    for pos in out:
        put(cache.k_pages, cache, 0, pos, 1, -INF, dim=3)
    got = cache.attend(q)
    cache.check_status()
    ref.assert_bounded(got[:1, :, 2:], want[:, :, 2:], bound[:, :, 2:])
    assert torch.isfinite(got).all()
