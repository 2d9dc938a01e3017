"""Argument checks of the rotation, paged-append and paged-attention entry points, made before
anything is launched: no GPU needed."""

import ctypes

import pytest
import torch

from attention_sinks_b200 import PagedKVCache, _lib, rope_frequencies, rotary

P = 4096  # a 16-byte aligned address that nothing reads


def paged(**kw):
    d = dict(k=P, v=P, table=P, lens=P, status=P, dtype=_lib.DTYPE_BF16, batch=2, heads_kv=2, head_dim=64, page_size=16,
             pages=10, table_width=4, pad_=0, table_stride=4, k_stride_p=2048, k_stride_h=1024, v_stride_p=2048,
             v_stride_h=1024)
    d.update(kw)
    return _lib.PagedKV(**d)


def rows(heads=2, n=1, dtype=_lib.DTYPE_BF16, data=P, sb=None, sh=64, st=64):
    return _lib.Rows(data, dtype, heads, n, 0, heads * 64 if sb is None else sb, sh, st)


def attention(lib, kv, q=None, shared=0, out=P, sb=256, sh=64, ws=P, nbytes=1 << 30):
    q = rows(heads=4) if q is None else q
    return lib.sink_paged_attention(ctypes.byref(q), ctypes.byref(kv), shared, 0.125, out, sb, sh, ws, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(k=None), _lib.EINVAL), (dict(table=None), _lib.EINVAL), (dict(lens=None), _lib.EINVAL),
    (dict(status=None), _lib.EINVAL), (dict(batch=0), _lib.EINVAL), (dict(pages=0), _lib.EINVAL),
    (dict(table_width=0), _lib.EINVAL), (dict(page_size=0), _lib.EINVAL), (dict(page_size=48), _lib.EINVAL),
    (dict(page_size=128, table_width=1 << 26), _lib.EINVAL), (dict(dtype=_lib.DTYPE_F32), _lib.EDTYPE),
    (dict(page_size=16, table_width=(1 << 27) - 1), _lib.EINVAL),  # rows end less than a chunk before 2^31
    (dict(dtype=9), _lib.EDTYPE), (dict(dtype=_lib.DTYPE_F16), _lib.EDTYPE), (dict(head_dim=96), _lib.EHEADDIM),
    (dict(head_dim=256), _lib.EHEADDIM), (dict(heads_kv=3), _lib.EGROUP), (dict(heads_kv=8), _lib.EGROUP),
    (dict(k=P + 2), _lib.ELAYOUT), (dict(v_stride_p=2044), _lib.ELAYOUT), (dict(k_stride_h=-1024), _lib.ELAYOUT),
])
def test_paged_attention_refusals(built_lib, change, code):
    assert attention(built_lib, paged(**change)) == code


def test_paged_attention_refuses_queries_and_prefixes(built_lib):
    lib = built_lib
    assert attention(lib, paged(), q=rows(heads=4, n=2)) == _lib.EINVAL
    assert attention(lib, paged(), q=rows(heads=18)) == _lib.EGROUP
    assert attention(lib, paged(), q=rows(heads=4, data=P + 8)) == _lib.ELAYOUT
    assert attention(lib, paged(), q=rows(heads=4, sh=65)) == _lib.ELAYOUT
    for shared in (-16, 8, 80):  # negative, not whole pages, more than the table holds
        assert attention(lib, paged(), shared=shared) == _lib.EINVAL
    assert attention(lib, paged(), out=None) == _lib.EINVAL
    assert attention(lib, paged(), ws=None) == _lib.EWORKSPACE
    assert attention(lib, paged(), nbytes=16) == _lib.EWORKSPACE


def test_workspace_is_host_arithmetic(built_lib):
    need = _lib.paged_workspace_bytes
    assert need(64, 8, 16, 128, 4096, 148) > 0
    for bad in ((0, 8, 16, 128, 0, 148), (1, 8, 12, 128, 0, 148), (1, 1, 9, 128, 0, 148), (1, 8, 16, 96, 0, 148),
                (1, 8, 16, 128, 0, 0), (1, 8, 16, 128, -128, 148), (1 << 23, 8, 16, 128, 0, 148)):
        assert need(*bad) == 0


def test_append_refusals(built_lib):
    def call(kv, k=None, v=None, q=None, q_out=None, rot=None):
        k, v = rows() if k is None else k, rows() if v is None else v
        ref = lambda x: ctypes.byref(x) if x is not None else None  # noqa: E731
        return built_lib.sink_paged_append(ctypes.byref(kv), ref(k), ref(v), None, ref(q), ref(q_out), ref(rot), None)

    assert call(paged(lens=None)) == _lib.EINVAL
    assert call(paged(), k=rows(heads=3)) == _lib.EINVAL
    assert call(paged(), v=rows(n=2)) == _lib.EINVAL
    assert call(paged(), k=rows(n=0), v=rows(n=0)) == _lib.EINVAL
    assert call(paged(), k=rows(dtype=_lib.DTYPE_F16)) == _lib.EDTYPE
    assert call(paged(), q=rows(heads=4)) == _lib.EINVAL  # nowhere to put it
    assert call(paged(), q=rows(heads=4), q_out=rows(heads=2)) == _lib.EINVAL
    assert call(paged(), rot=_lib.Rotation(P, 33, 0, 1.0, 0)) == _lib.EINVAL
    assert call(paged(), rot=_lib.Rotation(None, 32, 0, 1.0, 0)) == _lib.EINVAL
    assert call(paged(head_dim=1024), rot=None) == _lib.EHEADDIM
    big = 1 << 30
    assert call(paged(batch=4), k=rows(n=big), v=rows(n=big)) == _lib.EINVAL


def test_rotary_refusals(built_lib):
    def call(q=None, k=None, k_out=None, d=64, pos=P, rot=None, batch=1, q_out=None):
        q = rows() if q is None else q
        ref = lambda x: ctypes.byref(x) if x is not None else None  # noqa: E731
        rot = _lib.Rotation(P, 32, 0, 1.0, 0) if rot is None else rot
        return built_lib.sink_rotary(batch, d, ref(q), ref(q if q_out is None else q_out), ref(k), ref(k_out), pos, 0,
                                     ref(rot), None)

    assert call(batch=0) == _lib.EINVAL
    assert call(pos=None) == _lib.EINVAL
    assert call(k=rows()) == _lib.EINVAL
    assert call(k=rows(n=3), k_out=rows(n=3)) == _lib.EINVAL
    assert call(k=rows(dtype=_lib.DTYPE_F16), k_out=rows(dtype=_lib.DTYPE_F16)) == _lib.EDTYPE
    assert call(q=rows(dtype=7)) == _lib.EDTYPE
    assert call(q_out=rows(heads=1)) == _lib.EINVAL
    assert call(d=600) == _lib.EHEADDIM
    assert call(rot=_lib.Rotation(P, 64, 0, 1.0, 0)) == _lib.EINVAL
    assert call(rot=_lib.Rotation(P, -1, 0, 1.0, 0)) == _lib.EINVAL
    assert call(q=rows(n=1 << 30), batch=4) == _lib.EINVAL


def test_host_tensors_are_refused():
    f, _ = rope_frequencies(64)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary(torch.zeros(1, 2, 3, 64), None, torch.arange(3), f)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVCache(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32),
                     torch.zeros(1, dtype=torch.int32))


def test_rope_frequencies():
    f, a = rope_frequencies(8, base=100.0)
    assert a == 1.0 and f.dtype == torch.float64
    torch.testing.assert_close(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    torch.testing.assert_close(rope_frequencies(8, 100.0, "linear", 4.0)[0], f / 4)
    ntk = rope_frequencies(64, kind="ntk", factor=1.0, original_length=4096, length=16384)[0]
    plain = rope_frequencies(64)[0]
    # the highest frequency stays, the lowest turns over 16,384 rows as it did over 4,096
    assert ntk[0] == plain[0]
    torch.testing.assert_close(ntk[-1] * 16384, plain[-1] * 4096)
    l3 = rope_frequencies(64, 500000.0, "llama3", 32.0, 8192)[0]
    base = rope_frequencies(64, 500000.0)[0]
    assert torch.equal(l3[:8], base[:8]) and torch.equal(l3[-4:], base[-4:] / 32)
    assert bool((l3[1:] < l3[:-1]).all())
    yarn, a = rope_frequencies(64, kind="yarn", factor=16.0, original_length=4096)
    assert abs(a - 1.2772588722239782) < 1e-12
    assert yarn[0] == plain[0] and torch.equal(yarn[-1:], plain[-1:] / 16)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, factor=0.5), dict(rot_dim=8, kind="other")):
        with pytest.raises(ValueError):
            rope_frequencies(**bad)


@pytest.fixture
def plain_launch(monkeypatch):
    """rotary's launch by the plain formula, on bare values as a kernel sees them."""
    from attention_sinks_b200 import rope
    from tests import op_reference

    def launch(q, k, positions, inv_freq, interleaved, scale, inverse):
        bare = [None if x is None else torch.autograd.forward_ad.unpack_dual(x).primal.detach() for x in (q, k)]
        return tuple(None if x is None else op_reference.rotate(x, positions, inv_freq, interleaved, scale,
                                                                -1 if inverse else 1).to(x.dtype) for x in bare)

    monkeypatch.setattr(rope, "_launch", launch)


@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_rotary_carries_tangents(plain_launch, which):
    from torch.autograd import forward_ad as fw

    from tests import op_reference
    g = torch.Generator().manual_seed(1)
    f, pos = rope_frequencies(8)[0], torch.arange(5) + 3
    q, k, tq, tk = (torch.randn(2, h, 5, 12, generator=g, dtype=torch.float64) for h in (3, 1, 3, 1))
    with fw.dual_level():
        x = fw.make_dual(q, tq) if which != "k" else q
        y = fw.make_dual(k, tk) if which != "q" else k
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                got = [fw.unpack_dual(z) for z in rotary(x, y, pos, f, True, 1.5)]
            for z, value, tangent, there in zip(got, (q, k), (tq, tk), (which != "k", which != "q")):
                torch.testing.assert_close(z.primal, op_reference.rotate(value, pos, f, True, 1.5))
                if there:
                    torch.testing.assert_close(z.tangent, op_reference.rotate(tangent, pos, f, True, 1.5))
                else:
                    assert z.tangent is None
        alone, none = rotary(x, None, pos, f)
        assert none is None and (fw.unpack_dual(alone).tangent is not None) == (which != "k")


def test_rotary_tangents_of_gradients(plain_launch):
    """Forward over reverse: |rotate(x)|^2 has the gradient 2 x, whose tangent is 2 t."""
    from torch.autograd import forward_ad as fw
    g = torch.Generator().manual_seed(2)
    f, pos = rope_frequencies(8)[0], torch.arange(5)
    q, k, t = (torch.randn(1, 2, 5, 8, generator=g, dtype=torch.float64) for _ in range(3))
    q.requires_grad_(True), k.requires_grad_(True)
    with fw.dual_level():
        for create in (True, False):
            a, b = rotary(fw.make_dual(q, t), k, pos, f)
            dq, dk = torch.autograd.grad((a * a).sum() + (b * b).sum(), (q, k), create_graph=create)
            torch.testing.assert_close(fw.unpack_dual(dq).tangent, 2 * t)
            torch.testing.assert_close(dk.detach(), 2 * k.detach())
            s = t.clone().requires_grad_(True)  # reverse over forward
            got = fw.unpack_dual(rotary(fw.make_dual(q, s), None, pos, f)[0]).tangent
            ds, = torch.autograd.grad((got * got).sum(), s)
            torch.testing.assert_close(ds, 2 * t)


def test_rotary_refuses_frequencies_that_ask_for_gradients(plain_launch):
    from torch.autograd import forward_ad as fw
    f, pos = rope_frequencies(8)[0], torch.arange(5)
    q = torch.ones(1, 2, 5, 8, dtype=torch.float64)
    learned = f.clone().requires_grad_(True)
    for x in (q, q.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="frequencies"):
            rotary(x, None, pos, learned)
    with torch.no_grad():
        torch.testing.assert_close(rotary(q, None, pos, learned)[0], rotary(q, None, pos, f)[0])
    with fw.dual_level(), pytest.raises(RuntimeError, match="frequencies"):
        rotary(q, None, pos, fw.make_dual(f, f))


def test_attributes_of_a_paged_cache_cannot_be_replaced():
    cache = PagedKVCache.__new__(PagedKVCache)  # attributes alone: a cache is made over CUDA tensors
    lens = cache.lens = torch.tensor([3, 4], dtype=torch.int32)
    cache.page_size = 16
    cache._fixed = frozenset(cache.__dict__)
    cache.lens += 1  # in place
    assert cache.lens is lens and lens.tolist() == [4, 5]
    with pytest.raises(AttributeError, match="in place"):
        cache.lens = cache.lens + 1
    with pytest.raises(AttributeError, match="in place"):
        cache.page_size = 32
    with pytest.raises(AttributeError, match="removed"):
        del cache.lens
    cache.name = "layer 3"  # a caller's own
    cache.name = "layer 4"
    del cache.name
    assert cache.lens is lens and cache.page_size == 16


def test_sizes_past_32_bits_are_refused_not_cut():
    for good in (0, -(1 << 31), (1 << 31) - 1):
        assert _lib.int32("x", good) == good
    for bad in (1 << 31, (1 << 32) + 16, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="32 bits"):
            _lib.int32("x", bad)
    for shape in ((1, 1, (1 << 32) + 1, 64), (1, (1 << 32) + 1, 1, 64)):
        with pytest.raises(ValueError, match="32 bits"):
            _lib.RowsArg(torch.empty(64, dtype=torch.bfloat16, device="meta").expand(shape))


def test_every_status_bit_is_reported():
    _lib.raise_status(0)
    page, wait = "page index outside", "bounded wait ran out"
    for status, there, absent in ((1, [wait], [page]), (2, [page], [wait]), (3, [page, wait], []),
                                  (4, ["unknown"], [page, wait]), (7, [page, wait, "unknown"], [])):
        with pytest.raises(RuntimeError, match=f"sinkcache_b200.*0x{status:x}") as e:
            _lib.raise_status(status)
        assert all(x in str(e.value) for x in there) and not any(x in str(e.value) for x in absent)


@pytest.mark.parametrize("factor,length,divisor", [(4.0, None, 13.0), (2.0, None, 3.0), (4.0, 16384, 13.0),
                                                   (4.0, 8192, 5.0), (4.0, 4096, 1.0), (4.0, 1000, 1.0),
                                                   (1.0, 16384, 4.0)])
def test_ntk_frequencies_as_documented(factor, length, divisor):
    """Highest frequency kept, lowest divided by factor * reach - (factor - 1); every frequency is the
    same power of the raised base."""
    f = rope_frequencies(64, 50000.0)[0]
    ntk, scaling = rope_frequencies(64, 50000.0, "ntk", factor, original_length=4096, length=length)
    assert scaling == 1.0 and ntk[0] == f[0]
    torch.testing.assert_close(f[-1] / ntk[-1], torch.tensor(divisor, dtype=torch.float64))
    torch.testing.assert_close(f / ntk, divisor ** (torch.arange(32, dtype=torch.float64) / 31))
    torch.testing.assert_close(rope_frequencies(2, kind="ntk", factor=4.0)[0], torch.ones(1, dtype=torch.float64))


@pytest.mark.parametrize("kind", ["linear", "llama3", "yarn", "dynamic"])
@pytest.mark.parametrize("length", [4096, 10000, 16384])
def test_frequencies_match_the_model_library(kind, length):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    params = {"rope_type": kind, "rope_theta": 50000.0, "factor": 4.0, "original_max_position_embeddings": 4096,
              "low_freq_factor": 1.0, "high_freq_factor": 4.0}
    c = LlamaConfig(hidden_size=1024, num_attention_heads=8, head_dim=128, max_position_embeddings=4096,
                    rope_parameters=params)
    want, scaling = ROPE_INIT_FUNCTIONS[kind](c, torch.device("cpu"), seq_len=length)
    f, a = rope_frequencies(128, 50000.0, "ntk" if kind == "dynamic" else kind, 4.0, 4096, length)
    # the library's are fp32: the exponent 2 i / 128, its power (ln 50000 = 10.8 times its rounding) and a
    # division or blend, some 16 units of 2^-24 in all
    torch.testing.assert_close(f, want.double(), rtol=16 * 2.0 ** -24, atol=0)
    assert abs(a - scaling) < 1e-6
