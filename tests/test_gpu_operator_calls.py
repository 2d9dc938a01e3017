"""Calls of the rotation and the paged cache that their documentation allows or refuses, one by
one: forward-mode derivatives, changed attributes, sizes past 32 bits."""

import pytest
import torch
from torch.autograd import forward_ad as fw

from attention_sinks_b200 import rope_frequencies, rotary
from tests import op_reference as ref
from tests.test_gpu_operators import BF, DEV, FP, gen, make_cache, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_rotary_tangents_match_the_formula(dtype):
    g, f = gen(41), rope_frequencies(48)[0].to(DEV)
    pos = torch.randint(0, 5000, (2, 21), generator=g, device=DEV)
    q, k, tq, tk = (randn(g, 2, h, 21, 80, dtype=dtype) for h in (4, 2, 4, 2))
    with fw.dual_level():
        both = rotary(fw.make_dual(q, tq), fw.make_dual(k, tk), pos, f, attention_scaling=1.25)
        one = rotary(q, fw.make_dual(k, tk), pos, f, attention_scaling=1.25)
        assert fw.unpack_dual(one[0]).tangent is None
        for got, x, t in ((both[0], q, tq), (both[1], k, tk), (one[1], k, tk)):
            got = fw.unpack_dual(got)
            for y, value in ((got.primal, x), (got.tangent, t)):
                want = ref.rotate(value, pos, f, False, 1.25)
                ref.assert_bounded(y, want, ref.rotate_bound(value, want, f, False, 1.25, dtype))


def test_rotary_tangents_match_differences():
    """The rotation is linear: (f(x + t) - f(x - t)) / 2 is the tangent but for fp32 rounding, of
    x +- t (2^-24 of them, turned by two terms) and of each rotation (its own bound)."""
    g, f = gen(42), rope_frequencies(8)[0].to(DEV)
    pos = torch.arange(3, device=DEV) + 11
    q, t = randn(g, 1, 2, 3, 8, dtype=FP), randn(g, 1, 2, 3, 8, dtype=FP)
    with fw.dual_level():
        got = fw.unpack_dual(rotary(fw.make_dual(q, t), None, pos, f)[0]).tangent
    diff = (rotary(q + t, None, pos, f)[0] - rotary(q - t, None, pos, f)[0]) / 2
    size = q.abs() + t.abs()
    bound = 2 * 2.0 ** -24 * (size + size.roll(4, -1)).double()
    for x in (q + t, q - t, t):
        bound += ref.rotate_bound(x, ref.rotate(x, pos, f), f, False, 1.0, FP)
    ref.assert_bounded(got, diff.double(), bound + 2.0 ** -24 * diff.abs())


def test_rotary_gradient_of_a_tangent():
    g, f = gen(43), rope_frequencies(64)[0].to(DEV)
    pos = torch.arange(20, device=DEV)
    q, t, w = (randn(g, 1, 2, 20, 64, dtype=FP) for _ in range(3))
    t.requires_grad_(True)
    with fw.dual_level():
        got = fw.unpack_dual(rotary(fw.make_dual(q, t), None, pos, f)[0]).tangent
        dt, = torch.autograd.grad(got, t, w)
    want = ref.rotate(w, pos, f, sign=-1)
    ref.assert_bounded(dt, want, ref.rotate_bound(w, want, f, False, 1.0, FP))


def test_the_paged_cache_refuses_tangents():
    g = gen(44)
    cache = make_cache(g, [40, 20], 2, 16, 64)
    q, k = randn(g, 2, 4, 1, 64), randn(g, 2, 2, 1, 64)
    with fw.dual_level():
        for bad in (lambda: cache.attend(fw.make_dual(q, q)), lambda: cache.append(fw.make_dual(k, k), k),
                    lambda: cache.append(k, fw.make_dual(k, k)),
                    lambda: cache.append(k, k, q=fw.make_dual(q, q))):
            with pytest.raises(RuntimeError, match="tangents"):
                bad()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangents"):
                bad()
        want = cache.attend(q)  # a level alone is nothing to refuse
        assert torch.equal(cache.attend(fw.unpack_dual(fw.make_dual(q, q)).primal), want)


def test_the_paged_cache_keeps_its_tensors():
    g = gen(45)
    cache = make_cache(g, [40, 20], 2, 16, 64)
    q = randn(g, 2, 4, 1, 64)
    want = cache.attend(q)
    for name in ("k_pages", "v_pages", "block_table", "lens", "status"):
        with pytest.raises(AttributeError, match="in place"):
            setattr(cache, name, getattr(cache, name).clone())
    cache.lens -= 1
    want_less, bound = ref.attend(q, cache.k_pages, cache.v_pages, cache.block_table, cache.lens, 0.125)
    ref.assert_bounded(cache.attend(q), want_less, bound)
    cache.lens += 1
    assert torch.equal(cache.attend(q), want)


def test_sizes_past_32_bits_are_refused_not_cut():
    g = gen(46)
    cache = make_cache(g, [40, 20], 2, 16, 64)
    q = randn(g, 2, 4, 1, 64)
    for shared in (1 << 32, (1 << 32) + 16, -(1 << 32)):
        with pytest.raises(ValueError, match="32 bits"):
            cache.attend(q, shared_len=shared)
    many = randn(g, 2, 2, 1, 64).expand(2, 2, (1 << 32) + 1, 64)  # one row seen as 2^32 + 1
    before = cache.v_pages.clone()
    with pytest.raises(ValueError, match="32 bits"):
        cache.append(many, many)
    assert torch.equal(cache.v_pages.view(torch.int16), before.view(torch.int16))


def test_two_sequences_that_append_to_one_slot():
    """Each value of the slot is one sequence's or the other's, and nothing else moves."""
    g = gen(47)
    cache = make_cache(g, [40, 40, 20], 2, 16, 64, fill=0.0)
    cache.block_table[1, 2] = cache.block_table[0, 2]
    k, v = randn(g, 3, 2, 4, 64), randn(g, 3, 2, 4, 64)
    before = [x.clone() for x in (cache.k_pages, cache.v_pages)]
    cache.append(k, v)
    cache.check_status()
    page = int(cache.block_table[0, 2])
    for pages, was, new in zip((cache.k_pages, cache.v_pages), before, (k, v)):
        got = pages[page, :, 4:8]
        assert bool(((got == new[0]) | (got == new[1])).all())
        was[page, :, 4:8] = got
        own = int(cache.block_table[2, 1])
        was[own, :, 0:4] = new[2]
        assert torch.equal(pages, was)
