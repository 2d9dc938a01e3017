"""The paged attention's bounded waits, made to run out: the library's test hook
(sink_debug_fail_next_wait) leaves one tile of keys or values of every CTA unissued -- no copy, no
arrival -- with the waits of that launch bounded to a few thousand polls.  The CTAs give up, wait
for what they did issue, free their tensor memory and set SINK_STATUS_WAIT_TIMEOUT; the next call
on the same cache is right."""

import pytest
import torch

from attention_sinks_b200 import _lib
from tests import op_reference as ref
from tests.test_gpu_operators import DEV, gen, make_cache, randn

pytestmark = pytest.mark.gpu
POLLS = 4096

# 13 chunks or more for every CTA of a device of 148 SMs, in each kind of work
KINDS = {"own": (8, 16, 8, 128, 0, 4000), "own of 64 dims": (8, 16, 8, 64, 0, 4000),
         "wide prefix, pair of tiles": (70, 32, 8, 128, 16384, 40),
         "narrow prefix": (2, 16, 8, 64, 32768, 300)}


@pytest.fixture(scope="module", params=KINDS, ids=list(KINDS))
def case(request):
    batch, hq, hkv, d, shared, own = KINDS[request.param]
    g = gen(batch + d)
    cache = make_cache(g, [shared + own - i % 30 for i in range(batch)], hkv, 128, d, shared=shared)
    q = randn(g, batch, hq, 1, d)
    want = cache.attend(q, shared_len=shared)
    cache.check_status()
    lo = range(0, batch, max(1, batch // 8))  # some sequences against the formula
    some = torch.tensor(list(lo), device=DEV)
    table = cache.block_table[some]
    table[:, :shared // 128] = cache.block_table[0, :shared // 128]
    exact, bound = ref.attend(q[some], cache.k_pages, cache.v_pages, table, cache.lens[some], d ** -0.5)
    ref.assert_bounded(want[some], exact, bound)
    return cache, q, shared, want


@pytest.mark.parametrize("tile", [0, 1, 2, 3, 4, 5, 9, 10, 11, 12, 13, 20, 21])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(case, tile):
    cache, q, shared, want = case
    _lib.fail_next_wait(tile, POLLS)
    cache.attend(q, shared_len=shared)
    with pytest.raises(RuntimeError, match="bounded wait ran out"):
        cache.check_status()
    for _ in range(3):
        assert torch.equal(cache.attend(q, shared_len=shared), want)
    cache.check_status()


def test_ctas_without_the_tile_run_normally():
    g = gen(50)
    cache = make_cache(g, [200, 130], 2, 64, 64)
    q = randn(g, 2, 4, 1, 64)
    want = cache.attend(q)
    _lib.fail_next_wait(1000, 1 << 20)
    assert torch.equal(cache.attend(q), want)
    cache.check_status()


def test_a_run_out_wait_and_a_bad_page_are_both_reported():
    g = gen(51)
    cache = make_cache(g, [4000, 500], 8, 64, 64)
    q = randn(g, 2, 16, 1, 64)
    want = cache.attend(q)
    page = int(cache.block_table[1, 0])
    cache.block_table[1, 0] = -7
    _lib.fail_next_wait(3, POLLS)
    cache.attend(q)
    with pytest.raises(RuntimeError, match="bounded wait ran out.*page index outside"):
        cache.check_status()
    cache.block_table[1, 0] = page
    assert torch.equal(cache.attend(q), want)
    cache.check_status()


def test_a_call_that_is_refused_leaves_the_hook_armed():
    g = gen(52)
    cache = make_cache(g, [4000, 3000], 8, 64, 64)
    q = randn(g, 2, 16, 1, 64)
    want = cache.attend(q)
    _lib.fail_next_wait(0, POLLS)
    with pytest.raises(RuntimeError, match="sinkcache_b200"):
        cache.attend(q, shared_len=8)
    cache.attend(q)
    with pytest.raises(RuntimeError, match="bounded wait"):
        cache.check_status()
    assert torch.equal(cache.attend(q), want)
