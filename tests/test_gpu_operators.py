"""The rotation, paged-append and shared-prefix attention kernels against 64-bit plain
implementations (tests/op_reference.py), with bounds counted from the types' roundings."""

import pytest
import torch

from attention_sinks_b200 import PagedKVCache, _lib, apply_rope, rope_frequencies, rotary
from tests import op_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=BF):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


# ------------------------------------------------------------------------------- rotation


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "inter"])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 32), (80, 80), (96, 36), (6, 2), (256, 64), (17, 6), (512, 512)])
@pytest.mark.parametrize("b,t", [(1, 1), (2, 17), (3, 64), (1, 130)])
def test_rotary_matches_the_formula(dtype, interleaved, d, rot, b, t):
    g = gen(d * 7 + t)
    q, k = randn(g, b, 6, t, d, dtype=dtype), randn(g, b, 2, t, d, dtype=dtype)
    f, _ = rope_frequencies(rot)
    pos = torch.randint(0, 1 << 20, (b, t), generator=g, device=DEV)
    scaling = 1.0 if t % 2 else 1.25
    got = rotary(q, k, pos, f.to(DEV), interleaved=interleaved, attention_scaling=scaling)
    for x, y in zip((q, k), got):
        want = ref.rotate(x, pos, f, interleaved, scaling)
        assert y.dtype == dtype and y.shape == x.shape
        ref.assert_bounded(y, want, ref.rotate_bound(x, want, f, interleaved, scaling, dtype))
        assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_far_and_negative_positions():
    f, _ = rope_frequencies(128, base=500000.0)
    pos = torch.tensor([0, 1, -1, -4096, (1 << 31) + 7, (1 << 40) + 3], device=DEV)
    q = randn(gen(1), 1, 4, 6, 128, dtype=FP)
    y, none = rotary(q, None, pos, f.to(DEV))
    assert none is None
    want = ref.rotate(q, pos, f)
    # fp64 itself loses 2^-53 of a 2^40 rad angle, twice (product, quarter turns): 2^-11.5
    slack = torch.tensor([0, 0, 0, 0, 2.0 ** -20, 2.0 ** -11], device=DEV)[:, None].double() * 4
    ref.assert_bounded(y, want, ref.rotate_bound(q, want, f, False, 1.0, FP) + slack)
    torch.testing.assert_close(y[:, :, 0], q[:, :, 0], rtol=0, atol=0)
    back, _ = rotary(y[:, :, :4], None, -pos[:4], f.to(DEV))
    torch.testing.assert_close(back, q[:, :, :4], rtol=0, atol=2.0 ** -20)


def test_rotary_agrees_with_apply_rope():
    f, _ = rope_frequencies(64)
    pos = torch.arange(50, device=DEV)
    q = randn(gen(3), 2, 3, 50, 64, dtype=FP)
    torch.testing.assert_close(rotary(q, None, pos, f.to(DEV))[0], apply_rope(q, pos, f.to(DEV)), rtol=0, atol=1e-4)


@pytest.mark.parametrize("layout", ["bthd", "heads_of_qkv", "offset", "expanded", "d_strided"])
def test_rotary_takes_any_strides(layout):
    g, f = gen(5), rope_frequencies(64)[0]
    pos = torch.arange(33, device=DEV) + 5
    if layout == "bthd":
        q, k = randn(g, 2, 33, 4, 64).transpose(1, 2), randn(g, 2, 33, 2, 64).transpose(1, 2)
    elif layout == "heads_of_qkv":  # one projection's output, cut by heads
        qkv = randn(g, 2, 33, 8, 64).transpose(1, 2)
        q, k = qkv[:, :4], qkv[:, 4:6]
    elif layout == "offset":  # rows not 16-byte aligned
        q, k = randn(g, 2, 4, 33, 67)[..., 3:], randn(g, 2, 2, 33, 67)[..., 1:65]
    elif layout == "expanded":
        q, k = randn(g, 1, 1, 33, 64).expand(2, 4, 33, 64), randn(g, 2, 2, 1, 64).expand(2, 2, 33, 64)
    else:
        q, k = randn(g, 2, 4, 64, 33).transpose(2, 3), randn(g, 2, 2, 64, 33).transpose(2, 3)
    for x, y in zip((q, k), rotary(q, k, pos, f.to(DEV))):
        want = ref.rotate(x, pos, f)
        ref.assert_bounded(y, want, ref.rotate_bound(x, want, f, False, 1.0, BF))


@pytest.mark.parametrize("positions", ["int32", "strided", "one row", "column"])
def test_rotary_takes_any_positions(positions):
    g, f = gen(4), rope_frequencies(64)[0]
    q = randn(g, 2, 3, 10, 64)
    pos = torch.randint(0, 9999, (2, 10), generator=g, device=DEV)
    if positions == "int32":
        given = pos.to(torch.int32)
    elif positions == "strided":
        given = torch.stack((pos, pos + 1), -1).flatten(1)[:, ::2]
    elif positions == "one row":
        given, pos = pos[:1], pos[:1].expand(2, 10)
    else:
        given = pos.t().contiguous().t()
    y, _ = rotary(q, None, given, f)  # frequencies from the host are copied per call
    want = ref.rotate(q, pos, f)
    ref.assert_bounded(y, want, ref.rotate_bound(q, want, f, False, 1.0, BF))


def test_rotary_refusals():
    f = rope_frequencies(64)[0].to(DEV)
    q, pos = torch.zeros(2, 3, 5, 64, device=DEV), torch.arange(5, device=DEV)
    for bad in (lambda: rotary(q[0], None, pos, f), lambda: rotary(q, q[:1], pos, f),
                lambda: rotary(q, q.half(), pos, f), lambda: rotary(q, q[:, :, :4], pos, f),
                lambda: rotary(q, None, pos[:4], f), lambda: rotary(q, None, pos.float(), f),
                lambda: rotary(q, None, pos.cpu(), f), lambda: rotary(q, None, pos, torch.cat((f, f))),
                lambda: rotary(q, None, pos, f.view(2, 16)),
                lambda: rotary(torch.zeros(1, 1, 5, 1024, device=DEV), None, pos, f)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        rotary(q.double(), None, pos, f)


def test_rotary_empty_and_infinite():
    f = rope_frequencies(64)[0].to(DEV)
    q, k = rotary(torch.empty(2, 4, 0, 64, device=DEV), torch.empty(2, 1, 0, 64, device=DEV),
                  torch.empty(0, dtype=torch.long, device=DEV), f)
    assert q.shape == (2, 4, 0, 64) and k.shape == (2, 1, 0, 64)
    x = torch.ones(1, 1, 2, 64, device=DEV)
    x[0, 0, 0, 3] = float("nan")
    x[0, 0, 1, 40] = float("inf")
    y, _ = rotary(x, None, torch.tensor([9, 9], device=DEV), f)
    bad = ~torch.isfinite(y[0, 0])  # a pair spoils itself alone
    assert bad[0].nonzero().flatten().tolist() == [3, 35] and bad[1].nonzero().flatten().tolist() == [8, 40]


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "inter"])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_rotary_gradients_match_the_formula(interleaved, dtype):
    g, f = gen(7), rope_frequencies(48, kind="yarn", factor=8.0)[0]
    pos = torch.randint(0, 5000, (2, 21), generator=g, device=DEV)
    q = randn(g, 2, 21, 4, 80, dtype=dtype).transpose(1, 2).requires_grad_(True)
    k = randn(g, 2, 2, 21, 80, dtype=dtype).requires_grad_(True)
    qo, ko = rotary(q, k, pos, f.to(DEV), interleaved=interleaved, attention_scaling=1.5)
    dq, dk = randn(g, 2, 1, 21, 80, dtype=dtype).expand(2, 4, 21, 80), randn(g, 2, 2, 21, 80, dtype=dtype)
    got = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for dy, dx in zip((dq, dk), got):
        want = ref.rotate(dy, pos, f, interleaved, 1.5, sign=-1)
        ref.assert_bounded(dx, want, ref.rotate_bound(dy, want, f, interleaved, 1.5, dtype))


def test_rotary_gradients_match_differences_and_reach_one_side_alone():
    g, f = gen(8), rope_frequencies(8)[0].to(DEV)
    pos = torch.arange(3, device=DEV) + 11
    q, k = randn(g, 1, 2, 3, 8, dtype=FP), randn(g, 1, 1, 3, 8, dtype=FP)
    w = randn(g, 1, 2, 3, 8, dtype=FP)

    def loss(x):
        y = rotary(x, k, pos, f, attention_scaling=0.5)[0]
        return (w * y * y).sum()

    x = q.clone().requires_grad_(True)
    dx, = torch.autograd.grad(loss(x), x)
    # the loss is quadratic in x: central differences are exact but for the losses' rounding,
    # 48 terms of size up to 8 each way, 2^-24 * 48 * 8 over the step 2 * 0.25
    for i in (0, 5, 13, 47):
        e = torch.zeros_like(q).view(-1)
        e[i] = 0.25
        e = e.view_as(q)
        diff = (loss(q + e) - loss(q - e)) / 0.5
        assert abs(diff.item() - dx.view(-1)[i].item()) <= 2.0 ** -24 * 48 * 8 * 2 / 0.5
    kk = k.clone().requires_grad_(True)
    dk, = torch.autograd.grad(rotary(q, kk, pos, f)[1].sum(), kk)
    want = ref.rotate(torch.ones_like(k), pos, f, sign=-1)
    ref.assert_bounded(dk, want, ref.rotate_bound(torch.ones_like(k), want, f, False, 1.0, FP))
    qq = q.clone().requires_grad_(True)  # the gradient of the gradient: the rotation itself
    dq, = torch.autograd.grad((rotary(qq, kk, pos, f)[0] ** 2).sum(), qq, create_graph=True)
    ddq, = torch.autograd.grad(dq.sum(), qq)
    torch.testing.assert_close(ddq, torch.full_like(q, 2.0), rtol=0, atol=2.0 ** -18)


def test_rotary_refuses_a_backward_pass_at_changed_positions():
    f = rope_frequencies(64)[0].to(DEV)
    pos = torch.arange(3, device=DEV)
    x = randn(gen(6), 1, 1, 3, 64, dtype=FP).requires_grad_(True)
    y, _ = rotary(x, None, pos, f)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="changed in place"):
        torch.autograd.grad(y.sum(), x)


def test_rotary_in_a_graph_with_its_backward():
    """Forward and backward captured, after eager passes over the same leaf whose graphs are gone
    (torch ties a living graph's leaf to the stream it was made on, which no capture may join)."""
    g, f = gen(9), rope_frequencies(64)[0].to(DEV)
    pos = torch.arange(20, device=DEV)
    x = randn(g, 1, 4, 20, 64, dtype=FP).requires_grad_(True)
    dy = randn(g, 1, 4, 20, 64, dtype=FP)
    eager, = torch.autograd.grad(rotary(x, None, pos, f)[0], x, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(rotary(x, None, pos, f)[0], x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = rotary(x, None, pos, f)
        dx, = torch.autograd.grad(y, x, dy)
    pos.add_(1000)
    graph.replay()
    want = ref.rotate(dy, pos, f, sign=-1)
    ref.assert_bounded(dx, want, ref.rotate_bound(dy, want, f, False, 1.0, FP))
    want = ref.rotate(x, pos, f)
    ref.assert_bounded(y, want, ref.rotate_bound(x, want, f, False, 1.0, FP))
    pos.sub_(1000)
    graph.replay()
    assert torch.equal(dx, eager)


@pytest.mark.parametrize("kind,extra", [("linear", {}), ("llama3", {}), ("yarn", {}), ("dynamic", {})])
def test_rope_frequencies_match_the_model_library(kind, extra):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    params = {"rope_type": kind, "rope_theta": 50000.0, "factor": 4.0, "original_max_position_embeddings": 4096,
              "low_freq_factor": 1.0, "high_freq_factor": 4.0}
    c = LlamaConfig(hidden_size=1024, num_attention_heads=8, head_dim=128, max_position_embeddings=4096,
                    rope_parameters=params)
    want, scaling = ROPE_INIT_FUNCTIONS[kind](c, torch.device("cpu"), seq_len=16384)
    f, a = rope_frequencies(128, 50000.0, "ntk" if kind == "dynamic" else kind, 4.0, 4096, 16384)
    torch.testing.assert_close(f.float(), want, rtol=2e-5, atol=0)
    assert abs(a - scaling) < 1e-6


# ------------------------------------------------------------------------------- the cache


def make_cache(g, lens, hkv, page, d, dtype=BF, shared=0, spare=2, fill=float("nan"), layout="plain", **kw):
    """A cache whose rows [0, lens[b]) are random and whose every other slot is `fill`; table
    entries past a sequence's pages are -1, so nothing may be read through them."""
    b = len(lens)
    ns = shared // page
    need = [max(0, -(-n // page) - ns) for n in lens]
    pages = ns + sum(need) + spare
    width = max([ns + 1] + [ns + n for n in need])
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(sum(lens) + b))
    table = torch.full((b, width), -1, dtype=torch.int32)
    table[:, :ns] = order[:ns]
    at = ns
    for i, n in enumerate(need):
        table[i, ns:ns + n] = order[at:at + n]
        at += n
    if layout == "plain":
        kp, vp = (torch.full((pages, hkv, page, d), fill, device=DEV, dtype=dtype) for _ in range(2))
    else:  # keys and values of a page side by side
        both = torch.full((pages, 2, hkv, page, d), fill, device=DEV, dtype=dtype)
        kp, vp = both[:, 0], both[:, 1]
    for i, n in enumerate(lens):
        for j in range(-(-n // page)):
            r = min(page, n - j * page)
            p = int(table[i, j])
            kp[p, :, :r] = randn(g, hkv, r, d, dtype=dtype)
            vp[p, :, :r] = randn(g, hkv, r, d, dtype=dtype)
    return PagedKVCache(kp, vp, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), **kw)


def check_attend(cache, q, shared=0, scale=None, what=""):
    got = cache.attend(q, scale=scale, shared_len=shared)
    cache.check_status()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, bound = ref.attend(q, cache.k_pages, cache.v_pages, cache.block_table, cache.lens, scale, shared)
    assert got.shape == want.shape and got.dtype == q.dtype
    ref.assert_bounded(got, want, bound, what)
    return got


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (8, 8, 64), (32, 8, 64), (3, 1, 128), (10, 2, 64), (28, 4, 128),
                                      (24, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_paged_attention_ragged(dtype, hq, hkv, d, page):
    g = gen(page + hq)
    lens = [1, 0, page - 1, page, page + 1, 127, 128, 129, 255, 300, 517, 2]
    cache = make_cache(g, lens, hkv, page, d, dtype)
    got = check_attend(cache, randn(g, len(lens), hq, 1, d, dtype=dtype) * 2)
    assert not got[1].any()


@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF, 16, 8, 128), (HF, 32, 8, 64), (BF, 6, 2, 128), (HF, 7, 1, 64),
                                            (BF, 5, 5, 64), (BF, 16, 2, 128)])
@pytest.mark.parametrize("batch", [1, 2, 33, 70])
@pytest.mark.parametrize("page,shared", [(16, 16), (16, 144), (64, 640), (128, 128), (32, 2080)])
def test_shared_prefix_attention(dtype, hq, hkv, d, batch, page, shared):
    g = gen(shared + batch)
    lens = [shared + (37 * i) % 150 for i in range(batch)]
    cache = make_cache(g, lens, hkv, page, d, dtype, shared=shared)
    cache.block_table[1:, :shared // page] = -1  # the shared part is read through row 0 alone
    check_attend(cache, randn(g, batch, hq, 1, d, dtype=dtype) * 2, shared)


def test_shared_prefix_sequences_inside_it_and_idle():
    g = gen(11)
    lens = [512, 0, 1, 511, 300, 129, 128, 513, 700, 0]
    cache = make_cache(g, [max(n, 512) if i in (0, 7, 8) else n for i, n in enumerate(lens)], 4, 64, 128, shared=512)
    check_attend(cache, randn(g, 10, 8, 1, 128), 512)
    cache.lens.zero_()
    assert not cache.attend(randn(g, 10, 8, 1, 128), shared_len=512).any()


def test_one_prefix_many_query_tiles():
    g = gen(12)
    lens = [1024 + i % 40 for i in range(200)]
    for hq, hkv, d in ((16, 2, 128), (7, 1, 64)):
        cache = make_cache(g, lens, hkv, 128, d, shared=1024)
        check_attend(cache, randn(g, 200, hq, 1, d), 1024, what=f"{hq}/{hkv}")


def test_paged_attention_long_own_rows():
    g = gen(13)
    cache = make_cache(g, [20000, 5, 9001], 2, 128, 128)
    check_attend(cache, randn(g, 3, 8, 1, 128))
    cache = make_cache(g, [33000], 1, 16, 64, HF)
    check_attend(cache, randn(g, 1, 8, 1, 64, dtype=HF))


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_paged_attention_scores_that_jump(dtype):
    """Scores that grow, chunk after chunk, by far more than the rescaling threshold, and a row
    far above all others: the running maximum moves within a split and between splits."""
    g = gen(14)
    cache = make_cache(g, [3000, 1500], 2, 64, 128, dtype, shared=1024)
    q = randn(g, 2, 4, 1, 128, dtype=dtype)
    for n, pos in enumerate((100, 400, 700, 1000, 1300)):
        page = cache.block_table[0, pos // 64].item()
        cache.k_pages[page, :, pos % 64] = (n + 1) * 1.5 * q[0, ::2, 0]
    for shared in (0, 1024):
        if shared == 0:
            cache.block_table[1, :16] = cache.block_table[0, :16]
        check_attend(cache, q, shared)


def test_paged_attention_nan_and_infinity():
    """What a sequence attends to spoils its own output alone; what lies past its length, nothing."""
    g = gen(15)
    cache = make_cache(g, [130, 131, 129], 1, 64, 64, fill=float("inf"))
    q = randn(g, 3, 2, 1, 64)
    page = cache.block_table[1, 2].item()
    cache.v_pages[page, 0, 2, 5] = float("nan")
    got = cache.attend(q)
    assert torch.isnan(got[1, 0, :, 5]).all() and torch.isfinite(got[1, 0, :, 6:]).all()
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_paged_attention_scales(scale):
    g = gen(16)
    cache = make_cache(g, [200, 77], 2, 32, 64, shared=64)
    check_attend(cache, randn(g, 2, 4, 1, 64) * 0.5, 64, scale=scale)


def test_paged_attention_strides_and_layouts():
    g = gen(17)
    cache = make_cache(g, [200, 77, 300], 2, 32, 128, layout="side by side")
    wide = randn(g, 3, 1, 6, 128)
    check_attend(cache, wide[:, :, 1:5].transpose(1, 2))                  # heads of a wider projection
    check_attend(cache, randn(g, 3, 4, 1, 131)[..., 3:])                  # rows not 16-byte aligned
    check_attend(cache, randn(g, 1, 4, 1, 128).expand(3, 4, 1, 128))      # one query for all
    table = torch.full((3, 64), -1, dtype=torch.int32, device=DEV)
    table[:, 5:5 + cache.block_table.shape[1]] = cache.block_table
    sub = PagedKVCache(cache.k_pages, cache.v_pages, table[:, 5:5 + cache.block_table.shape[1]], cache.lens)
    q = randn(g, 3, 4, 1, 128)
    assert torch.equal(sub.attend(q), cache.attend(q))


@pytest.mark.parametrize("shared", [0, 32])
def test_paged_attention_many_sequences(shared):
    """More sequences than the kernel has threads, idle ones among them."""
    g = gen(20 + shared)
    lens = [0 if i % 7 == 3 else shared + (i * 13) % 40 + 1 for i in range(1100)]
    cache = make_cache(g, lens, 1, 16, 64, shared=shared)
    check_attend(cache, randn(g, 1100, 2, 1, 64), shared)


def test_paged_attention_refusals():
    g = gen(27)
    cache = make_cache(g, [40, 20], 2, 16, 64)
    q, k = randn(g, 2, 4, 1, 64), randn(g, 2, 2, 1, 64)
    for bad in (lambda: cache.attend(q[:1]), lambda: cache.attend(q.half()), lambda: cache.attend(randn(g, 2, 4, 2, 64)),
                lambda: cache.attend(q.cpu()), lambda: cache.append(k, k[:1]), lambda: cache.append(q, k),
                lambda: cache.append(k, k, counts=torch.zeros(2, device=DEV)),
                lambda: cache.append(k, k, counts=torch.zeros(3, dtype=torch.int32, device=DEV)),
                lambda: cache.append(k, k, q=randn(g, 2, 4, 3, 64)),
                lambda: PagedKVCache(cache.k_pages, cache.v_pages[:1], cache.block_table, cache.lens),
                lambda: PagedKVCache(cache.k_pages, cache.v_pages, cache.block_table.long(), cache.lens),
                lambda: PagedKVCache(cache.k_pages, cache.v_pages, cache.block_table, cache.lens[:1]),
                lambda: PagedKVCache(cache.k_pages, cache.v_pages, cache.block_table, cache.lens.cpu()),
                lambda: PagedKVCache(cache.k_pages.transpose(2, 3), cache.v_pages.transpose(2, 3), cache.block_table,
                                     cache.lens),
                lambda: PagedKVCache(cache.k_pages, cache.v_pages, cache.block_table, cache.lens,
                                     inv_freq=torch.ones(33, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.attend(q, shared_len=8), lambda: cache.attend(q, shared_len=-16),
                lambda: cache.attend(q, shared_len=1 << 20), lambda: cache.attend(randn(g, 2, 3, 1, 64)),
                lambda: cache.attend(randn(g, 2, 18, 1, 64)), lambda: cache.attend(q, scale=float("nan")),
                lambda: make_cache(g, [4], 1, 16, 64, FP).attend(randn(g, 1, 1, 1, 64, dtype=FP)),
                lambda: make_cache(g, [4], 1, 16, 80).attend(randn(g, 1, 1, 1, 80)),
                lambda: make_cache(g, [4], 1, 48, 64).attend(randn(g, 1, 1, 1, 64))):
        with pytest.raises(RuntimeError, match="sinkcache_b200"):
            bad()
    with pytest.raises(RuntimeError, match="gradients"):
        cache.attend(q.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="gradients"):
        cache.append(k.clone().requires_grad_(True), k)
    with torch.no_grad():
        cache.attend(q.clone().requires_grad_(True))
    cache.check_status()


def test_paged_attention_refuses_tables_of_too_much_work():
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    heads = 64
    width = sms * (1 << 22) // heads + 1  # one chunk of 128 rows per page, one more than 2^22 of them per SM
    pools = torch.zeros(1, heads, 128, 64, device=DEV, dtype=BF)
    table = torch.zeros(1, width, dtype=torch.int32, device=DEV)
    lens = torch.ones(1, dtype=torch.int32, device=DEV)
    q = randn(gen(28), 1, heads, 1, 64)
    with pytest.raises(RuntimeError, match="sinkcache_b200"):
        PagedKVCache(pools, pools.clone(), table, lens).attend(q)
    out = PagedKVCache(pools, pools.clone(), table[:, :width - 1], lens).attend(q)
    assert out.shape == (1, 1, heads, 64) and not out.any()


def test_paged_calls_on_nothing():
    pools = torch.zeros(3, 2, 16, 64, device=DEV, dtype=BF)
    none = PagedKVCache(pools, pools.clone(), torch.zeros(0, 4, dtype=torch.int32, device=DEV),
                        torch.zeros(0, dtype=torch.int32, device=DEV))
    assert none.attend(torch.zeros(0, 4, 1, 64, device=DEV, dtype=BF)).shape == (0, 1, 4, 64)
    some = make_cache(gen(26), [40, 20], 2, 16, 64)
    before = some.k_pages.clone()
    q = some.append(*(torch.zeros(2, 2, 0, 64, device=DEV, dtype=BF) for _ in range(2)),
                    q=torch.zeros(2, 4, 0, 64, device=DEV, dtype=BF))
    assert q.shape == (2, 4, 0, 64) and torch.equal(some.k_pages.view(torch.int16), before.view(torch.int16))


def test_append_of_more_than_there_is():
    """Counts past the tokens given are those tokens, lengths below zero nothing."""
    g = gen(28)
    cache = make_cache(g, [40, 20, 20], 2, 16, 64, fill=0.0)
    k, v = randn(g, 3, 2, 4, 64), randn(g, 3, 2, 4, 64)
    cache.lens[2] = -3
    kept = ref.gather(cache.v_pages, cache.block_table[2], 20)
    cache.append(k, v, counts=torch.tensor([9, -2, 4], dtype=torch.int32, device=DEV))
    cache.check_status()
    assert torch.equal(ref.gather(cache.v_pages, cache.block_table[0], 40)[:, 36:], v[0].double())
    assert torch.equal(ref.gather(cache.v_pages, cache.block_table[2], 20), kept)
    assert not cache.attend(randn(g, 3, 4, 1, 64))[2].any()


def test_attend_from_two_threads_on_one_stream():
    import threading
    g = gen(29)
    caches = [make_cache(g, [1500 + 31 * i for i in range(16)], 8, 64, 128, shared=1024) for _ in range(2)]
    qs = [randn(g, 16, 16, 1, 128) for _ in range(2)]
    want = [c.attend(q, shared_len=1024) for c, q in zip(caches, qs)]
    wrong = []

    def work(i):
        for _ in range(200):
            if not torch.equal(caches[i].attend(qs[i], shared_len=1024), want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_paged_attention_repeats_bit_for_bit():
    g = gen(18)
    cache = make_cache(g, [1024 + 13 * i for i in range(40)], 4, 64, 128, shared=1024)
    q = randn(g, 40, 16, 1, 128)
    first = cache.attend(q, shared_len=1024)
    for _ in range(5):
        assert torch.equal(cache.attend(q, shared_len=1024), first)


def test_pages_past_32_bit_offsets():
    """A pool of more than 2^31 elements, the rows at its far end."""
    pages, page, d = (1 << 31) // (2 * 128 * 128) + 8, 128, 128
    kp = torch.empty(pages, 2, page, d, dtype=BF, device=DEV)
    vp = torch.empty_like(kp)
    table = torch.tensor([[pages - 1, pages - 3], [0, pages - 2]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([200, 150], dtype=torch.int32, device=DEV)
    f = rope_frequencies(128)[0].to(DEV)
    cache = PagedKVCache(kp, vp, table, lens, inv_freq=f)
    g = gen(19)
    k, v = randn(g, 2, 2, 200, d), randn(g, 2, 2, 200, d)
    q = cache.append(k, v, q=randn(g, 2, 4, 200, d), counts=lens.clone())
    pos = torch.arange(200, device=DEV)
    want = ref.rotate(k, pos, f)
    bound = ref.rotate_bound(k, want, f, False, 1.0, BF)
    for i, n in enumerate((200, 150)):
        got = ref.gather(kp, table[i], n)
        ref.assert_bounded(got, want[i, :, :n], bound[i, :, :n])
        assert torch.equal(ref.gather(vp, table[i], n), v[i, :, :n].double())
    check_attend(cache, q[:, :, 149:150].contiguous())


# ------------------------------------------------------------------------------- append


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "inter"])
@pytest.mark.parametrize("d,rot,page", [(128, 128, 16), (64, 48, 64), (80, 40, 7), (96, 36, 32), (128, 0, 128)])
@pytest.mark.parametrize("tokens", [1, 5, 70])
def test_append_matches_the_formula(dtype, interleaved, d, rot, page, tokens):
    g = gen(d + tokens + page)
    counts = [tokens, 0, max(1, tokens // 2), tokens, 1]
    lens = [tokens, 0, 40 + counts[2], 3 * page + tokens, 1]
    cache = make_cache(g, lens, 3, page, d, dtype, fill=7.0)
    f = rope_frequencies(rot)[0].to(DEV) if rot else None
    cache = PagedKVCache(cache.k_pages, cache.v_pages, cache.block_table, cache.lens, inv_freq=f,
                         interleaved=interleaved, attention_scaling=1.125)
    before_k, before_v = cache.k_pages.clone(), cache.v_pages.clone()
    k, v, q = (randn(g, 5, h, tokens, d, dtype=dtype) for h in (3, 3, 6))
    q_out = cache.append(k, v, q=q, counts=torch.tensor(counts, dtype=torch.int32, device=DEV))
    cache.check_status()
    pos = torch.tensor([[n - c + t for t in range(tokens)] for n, c in zip(lens, counts)], device=DEV)

    def turned(x):
        if not rot:
            return x.double(), torch.zeros_like(x, dtype=torch.float64)
        want = ref.rotate(x, pos, f, interleaved, 1.125)
        return want, ref.rotate_bound(x, want, f, interleaved, 1.125, dtype)

    wk, bk = turned(k)
    wq, bq = turned(q)
    for i, c in enumerate(counts):
        ref.assert_bounded(q_out[i, :, :c], wq[i, :, :c], bq[i, :, :c]) if c else None
        assert not q_out[i, :, c:].any()
        for t in range(c):
            p = int(pos[i, t])
            at = int(cache.block_table[i, p // page]), p % page
            ref.assert_bounded(cache.k_pages[at[0], :, at[1]], wk[i, :, t], bk[i, :, t])
            assert torch.equal(cache.v_pages[at[0], :, at[1]], v[i, :, t])
            before_k[at[0], :, at[1]] = cache.k_pages[at[0], :, at[1]]
            before_v[at[0], :, at[1]] = v[i, :, t]
    assert torch.equal(cache.k_pages, before_k) and torch.equal(cache.v_pages, before_v)  # nothing else moved


def test_append_without_counts_or_query_and_with_strides():
    g = gen(21)
    f = rope_frequencies(64)[0].to(DEV)
    cache = make_cache(g, [40, 9, 8], 2, 16, 64, layout="side by side", inv_freq=f)
    kv = randn(g, 3, 8, 4, 64).transpose(1, 2)
    assert cache.append(kv[:, :2], kv[:, 2:]) is None
    pos = cache.lens[:, None] - 8 + torch.arange(8, device=DEV)
    want = ref.rotate(kv[:, :2], pos, f)
    bound = ref.rotate_bound(kv[:, :2], want, f, False, 1.0, BF)
    for i, n in enumerate((40, 9, 8)):
        ref.assert_bounded(ref.gather(cache.k_pages, cache.block_table[i], n)[:, n - 8:], want[i], bound[i])
        assert torch.equal(ref.gather(cache.v_pages, cache.block_table[i], n)[:, n - 8:], kv[i, 2:].double())


def test_bad_pages_are_reported_not_touched():
    g = gen(22)
    cache = make_cache(g, [40, 20], 2, 16, 64, fill=0.0)
    good = cache.k_pages.clone()
    table = cache.block_table.clone()
    q, k = randn(g, 2, 4, 1, 64), randn(g, 2, 2, 1, 64)
    whole = cache.attend(q)
    for bad in (-1, -5, cache.k_pages.shape[0], 1 << 30):
        cache.block_table.copy_(table)
        cache.block_table[0, 2] = bad
        got = cache.attend(q)
        assert torch.equal(got[1], whole[1])  # the other sequence is as it was
        with pytest.raises(RuntimeError, match="page"):
            cache.check_status()
        cache.check_status()  # once
        cache.append(k[:1].expand(2, 2, 1, 64), k, counts=torch.tensor([1, 0], dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="page"):
            cache.check_status()
        assert torch.equal(cache.k_pages, good)
    cache.block_table.copy_(table)
    cache.lens[0] = 16 * cache.block_table.shape[1] + 1  # past the table
    cache.attend(q)
    with pytest.raises(RuntimeError, match="page"):
        cache.check_status()
    cache.lens.copy_(torch.tensor([40, 20], dtype=torch.int32))
    assert torch.equal(cache.attend(q), whole)
    cache.check_status()


# ------------------------------------------------------------------------ together, in use


def test_prefill_then_decode_steps_in_a_graph():
    """A prompt appended once, a batch decoding from it: append and attend of every step from
    one captured graph, lengths advanced on the device, against the 64-bit formula."""
    g = gen(30)
    b, hq, hkv, d, page, prompt = 5, 8, 4, 128, 16, 48
    f, a = rope_frequencies(d, kind="llama3", factor=8.0)
    f = f.to(DEV)
    pages = prompt // page + 4 * b
    kp, vp = (torch.full((pages, hkv, page, d), float("nan"), device=DEV, dtype=BF) for _ in range(2))
    table = torch.full((b, prompt // page + 4), -1, dtype=torch.int32, device=DEV)
    table[:, :3] = torch.arange(3, device=DEV)
    table[:, 3:] = torch.arange(3, pages, device=DEV).view(b, 4)
    lens = torch.full((b,), prompt, dtype=torch.int32, device=DEV)
    cache = PagedKVCache(kp, vp, table, lens, inv_freq=f, attention_scaling=a)
    one = PagedKVCache(kp, vp, table[:1], lens[:1], inv_freq=f, attention_scaling=a, status=cache.status)
    k0, v0 = randn(g, 1, hkv, prompt, d), randn(g, 1, hkv, prompt, d)
    one.append(k0, v0)
    ks, vs = [k0.expand(b, hkv, prompt, d)], [v0.expand(b, hkv, prompt, d)]
    k, v, q = randn(g, b, hkv, 1, d), randn(g, b, hkv, 1, d), randn(g, b, hq, 1, d)
    graph = torch.cuda.CUDAGraph()

    def step():
        lens.add_(1)
        turned = cache.append(k, v, q=q)
        return turned, cache.attend(turned, shared_len=prompt)

    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        turned, out = step()
    assert int(lens[0]) == prompt  # capturing ran nothing
    for n in range(20):
        for x in (k, v, q):
            x.copy_(randn(g, *x.shape))
        ks.append(k.clone()), vs.append(v.clone())
        graph.replay()
        cache.check_status()
        assert lens.tolist() == [prompt + n + 1] * b
        want = ref.rotate(q, lens[:, None].long() - 1, f, scaling=a)
        ref.assert_bounded(turned, want, ref.rotate_bound(q, want, f, False, a, BF))
        want, bound = ref.attend(turned, kp, vp, table, lens, d ** -0.5, prompt)
        ref.assert_bounded(out, want, bound, f"step {n}")
    # the whole of it from the unrotated inputs: keys rounded to bf16 once after the rotation
    allk, allv = torch.cat(ks, 2), torch.cat(vs, 2)
    rk = ref.rotate(allk, torch.arange(allk.shape[2], device=DEV), f, scaling=a)
    for i in range(b):
        got = ref.gather(kp, table[i], prompt + 20)
        bound = ref.rotate_bound(allk[i:i + 1], rk[i:i + 1], f, False, a, BF)[0]
        ref.assert_bounded(got, rk[i], bound)
        assert torch.equal(ref.gather(vp, table[i], prompt + 20), allv[i].double())


def test_calls_on_two_streams_and_two_graphs():
    """Attention calls that run at the same time use scratch of their own: two streams, and two
    captured graphs replayed on them."""
    g = gen(31)
    caches = [make_cache(g, [2048 + 31 * i for i in range(24)], 8, 64, 128, shared=1024) for _ in range(2)]
    qs = [randn(g, 24, 16, 1, 128) for _ in range(2)]
    want = [c.attend(q, shared_len=1024) for c, q in zip(caches, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        outs = []
        for c, q, s in zip(caches, qs, streams):
            with torch.cuda.stream(s):
                outs.append(c.attend(q, shared_len=1024))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
    graphs, outs = [], []
    for c, q in zip(caches, qs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c.attend(q, shared_len=1024))
    for _ in range(10):
        for x in outs:
            x.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_layers_share_table_lengths_and_status():
    g = gen(32)
    first = make_cache(g, [100, 37], 2, 32, 64)
    second = PagedKVCache(torch.randn_like(first.k_pages.nan_to_num(0)), torch.randn_like(first.v_pages.nan_to_num(0)),
                          first.block_table, first.lens, status=first.status)
    q = randn(g, 2, 4, 1, 64)
    check_attend(second, q)
    second.block_table[1, 0] = 999
    second.attend(q)
    with pytest.raises(RuntimeError, match="page"):
        first.check_status()


def test_every_call_launches_the_library():
    g = gen(33)
    f = rope_frequencies(64)[0].to(DEV)
    cache = make_cache(g, [100, 37], 2, 32, 64, inv_freq=f)
    for call in (lambda: rotary(randn(g, 1, 2, 3, 64), None, torch.arange(3, device=DEV), f),
                 lambda: cache.append(randn(g, 2, 2, 1, 64), randn(g, 2, 2, 1, 64)),
                 lambda: cache.attend(randn(g, 2, 4, 1, 64))):
        before = _lib.launch_count()
        call()
        assert _lib.launch_count() > before
