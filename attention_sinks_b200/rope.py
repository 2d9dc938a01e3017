"""RoPE helpers in the Transformers (Llama / Qwen) half-split convention.

Dimension i of a head of size d pairs with i + d/2 and the pair is rotated by
pos * inv_freq[i]:  rope(x, p) = x * cos(p * theta) + rotate_half(x) * sin(p * theta).
Rotations compose by adding angles, so a key rotated at position p and then by -delta is
the key rotated at p - delta: that is what lets the sink cache move kept keys to new
positions after an eviction (src/sinkcache/rope.py:1-14).

The host-side helpers of the package: `rope_cos_sin` builds the fp32 cos/sin tables the
eviction kernel consumes (one [head_dim] table per shift), exactly as
src/sinkcache/rope.py:24-28 does; `apply_rope` / `rerotate` keep the reference's public
helpers (src/sinkcache/rope.py:43-54) for users and tests.

`rotary` is the rotation on the GPU: q and k in one kernel launch, half-split or interleaved
pairs, a part of the head, fp64 angles, with its backward pass.  `rope_frequencies` gives the
frequencies it takes, scaled for long contexts where asked.
"""

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    """(x1, x2) -> (-x2, x1) over the last dim (src/sinkcache/rope.py:19-21)."""
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat((-x2, x1), dim=-1)


def rope_cos_sin(positions: torch.Tensor, inv_freq: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 cos/sin of shape [..., rot_dim] for integer positions, as HF computes them
    (src/sinkcache/rope.py:24-28): angles = position * inv_freq in fp32, both halves equal."""
    freqs = positions.to(torch.float32)[..., None] * inv_freq.to(torch.float32)
    emb = torch.cat((freqs, freqs), dim=-1)
    return emb.cos(), emb.sin()


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate the first cos.shape[-1] dims of x in fp32, round once to x.dtype
    (src/sinkcache/rope.py:31-40)."""
    rot_dim = cos.shape[-1]
    xf = x.to(torch.float32)
    x_rot, x_pass = xf[..., :rot_dim], xf[..., rot_dim:]
    out = x_rot * cos + rotate_half(x_rot) * sin
    if x_pass.shape[-1]:
        out = torch.cat((out, x_pass), dim=-1)
    return out.to(x.dtype)


def apply_rope(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor) -> torch.Tensor:
    """Rotate x [batch, heads, seq, head_dim] at `positions` [seq] (src/sinkcache/rope.py:43-46)."""
    cos, sin = rope_cos_sin(positions.to(x.device), inv_freq.to(x.device))
    return _rotate(x, cos, sin)


def rerotate(keys: torch.Tensor, delta: int, inv_freq: torch.Tensor) -> torch.Tensor:
    """Shift already-rotated keys `delta` positions earlier: a rotation by -delta
    (src/sinkcache/rope.py:49-54)."""
    cos, sin = rope_cos_sin(torch.tensor(-delta, device=keys.device), inv_freq.to(keys.device))
    return _rotate(keys, cos, sin)


# ------------------------------------------------------------------ rotation on the GPU


def rope_frequencies(rot_dim: int, base: float = 10000.0, kind: str = "default", factor: float = 1.0,
                     original_length: int = 8192, length: int | None = None, low_freq_factor: float = 1.0,
                     high_freq_factor: float = 4.0, beta_fast: float = 32.0,
                     beta_slow: float = 1.0) -> tuple[torch.Tensor, float]:
    """(float64 inverse frequencies [rot_dim / 2], attention scaling) of a rotary embedding.

    base ** (-2i / rot_dim), then, for contexts `factor` times the `original_length` the model
    was trained on:
      "linear"   every frequency divided by factor (positions interpolated);
      "ntk"      the base multiplied by (factor * reach - (factor - 1)) ** (rot_dim / (rot_dim - 2)),
                 reach = length / original_length, at least 1: the highest frequency stays and the
                 lowest is divided by factor * reach - (factor - 1).  `length` is the context to be
                 served, original_length * factor when not given (a lowest frequency divided by
                 factor**2 - factor + 1); factor 1 divides by reach alone;
      "llama3"   wavelengths above original_length / low_freq_factor divided by factor, those
                 below original_length / high_freq_factor kept, a linear blend between;
      "yarn"     pairs that turn more than beta_fast times over the original length kept, those
                 that turn less than beta_slow times divided by factor, a ramp over the pair
                 index between; attention scaling 0.1 ln(factor) + 1."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be a positive even number, got {rot_dim}")
    if factor < 1.0:
        raise ValueError(f"a context is extended by a factor of 1 or more, got {factor}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    f = base ** (-i / rot_dim)
    if kind == "default":
        return f, 1.0
    if kind == "linear":
        return f / factor, 1.0
    if kind == "ntk":
        reach = max(length if length is not None else factor * original_length, original_length) / original_length
        if rot_dim == 2:
            return f, 1.0
        raised = base * (factor * reach - (factor - 1.0)) ** (rot_dim / (rot_dim - 2))
        return raised ** (-i / rot_dim), 1.0
    if kind == "llama3":
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        return f * keep + f / factor * (1.0 - keep), 1.0
    if kind == "yarn":
        def pair_turning(turns):  # the (fractional) pair that turns so often over the original length
            return rot_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_turning(beta_fast)), 0)
        high = min(math.ceil(pair_turning(beta_slow)), rot_dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return f * (1.0 - ramp) + f / factor * ramp, (0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
    raise ValueError(f"unknown kind of frequency scaling {kind!r}")


def rotation(inv_freq: torch.Tensor, interleaved: bool, scale: float, inverse: bool = False) -> "_lib.Rotation":
    return _lib.Rotation(inv_freq.data_ptr(), inv_freq.numel(), int(interleaved), float(scale), int(inverse))


def device_frequencies(inv_freq: torch.Tensor, device: torch.device) -> torch.Tensor:
    """`inv_freq` as the kernels read it: contiguous float64 on `device` (itself, if it is that)."""
    if inv_freq.dim() != 1:
        raise ValueError(f"inv_freq is one-dimensional, got {tuple(inv_freq.shape)}")
    return inv_freq.detach().to(device, torch.float64).contiguous()


class _RotaryCall:
    """A checked form of `rotary` call, with the descriptors of its tensors."""

    def __init__(self, q, k, positions, inv_freq):
        if q.dim() != 4:
            raise ValueError(f"q is [B, H, T, D], got {tuple(q.shape)}")
        device = q.device
        _lib.check_device(device)
        _lib.dtype_code(q.dtype)
        b, _, t, d = q.shape
        if k is not None and (k.dim() != 4 or k.shape[0] != b or k.shape[2] != t or k.shape[3] != d
                              or k.dtype != q.dtype or k.device != device):
            raise ValueError(f"k {tuple(k.shape)} {k.dtype} {k.device} does not go with q {tuple(q.shape)} {q.dtype} "
                             f"{device}")
        if positions.device != device or positions.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"positions are whole numbers on {device}, got {positions.dtype} on {positions.device}")
        if positions.shape not in ((t,), (b, t), (1, t)):
            raise ValueError(f"positions are [{t}] or [{b}, {t}], got {tuple(positions.shape)}")
        if inv_freq.dim() != 1 or 2 * inv_freq.numel() > d or d > 512:
            raise ValueError(f"inv_freq {tuple(inv_freq.shape)} is not one-dimensional, or rotates more than a head of "
                             f"{d} dims (at most 512)")
        self.device, self.index = device, device.index
        self.batch, self.dim = _lib.int32("batch", b), d
        # what a call has to convert first
        self.copy_q = q.stride(-1) != 1
        self.copy_k = k is not None and k.stride(-1) != 1
        self.copy_positions = positions.dtype != torch.int64 or (t > 1 and positions.stride(-1) != 1)
        self.copy_freq = inv_freq.dtype != torch.float64 or inv_freq.device != device or not inv_freq.is_contiguous()
        self.empty = not (q.numel() or (k is not None and k.numel()))
        like = _lib.layout_of(q, self.copy_q)
        self.q, self.q_out = _lib.RowsArg(like), _lib.RowsArg(torch.empty_like(like))
        if k is not None:
            like = _lib.layout_of(k, self.copy_k)
            self.k, self.k_out = _lib.RowsArg(like), _lib.RowsArg(torch.empty_like(like))
        several = positions.dim() == 2 and positions.shape[0] > 1
        self.pos_stride = 0 if not several else t if self.copy_positions else positions.stride(0)
        self.rot = _lib.Rotation(0, inv_freq.numel(), 0, 1.0, 0)
        self.rot_ref = ctypes.byref(self.rot)

    def __call__(self, q, k, positions, inv_freq, interleaved, scale, inverse):
        if _lib.current_device() != self.index:
            with torch.cuda.device(self.index):
                return self(q, k, positions, inv_freq, interleaved, scale, inverse)
        if self.copy_q:
            q = q.contiguous()
        if self.copy_k:
            k = k.contiguous()
        q_out = torch.empty_like(q)
        k_out = None if k is None else torch.empty_like(k)
        if self.empty:
            return q_out, k_out
        if self.copy_positions:
            positions = positions.to(torch.int64).contiguous()
        if self.copy_freq:
            inv_freq = device_frequencies(inv_freq, self.device)
        rot = self.rot
        rot.inv_freq, rot.interleaved, rot.scale, rot.inverse = inv_freq.data_ptr(), interleaved, scale, inverse
        rc = _lib.lib().sink_rotary(self.batch, self.dim, self.q.at(q), self.q_out.at(q_out),
                                    None if k is None else self.k.at(k),
                                    None if k is None else self.k_out.at(k_out), positions.data_ptr(),
                                    self.pos_stride, self.rot_ref, _lib.raw_stream(self.index))
        if rc:
            _lib._check(rc, "sink_rotary")
        return q_out, k_out


def _launch(q, k, positions, inv_freq, interleaved, scale, inverse):
    form = (_lib.form_of(q), _lib.form_of(k), _lib.form_of(positions), _lib.form_of(inv_freq))
    known = _lib.forms("rotary")
    call = known.get(form)
    if call is None:
        call = known[form] = _RotaryCall(q, k, positions, inv_freq)
    return call(q, k, positions, inv_freq, interleaved, scale, inverse)


class _Rotary(torch.autograd.Function):
    """The rotation is linear and (up to the attention scaling) orthogonal, so its backward
    pass is the rotation of the gradients by the negative angles: the same kernel, and itself
    differentiable.  Tangents are rotated as their tensors are."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, scale, inverse):
        ctx.set_materialize_grads(False)
        # neither is differentiable, so they need no saved-tensor hooks; their versions are
        # compared in the backward pass, as torch does for saved tensors
        ctx.kept = positions, inv_freq, positions._version, inv_freq._version
        ctx.how = interleaved, scale, inverse
        q_out, k_out = _launch(q, k, positions, inv_freq, interleaved, scale, inverse)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    def backward(ctx, dq, dk=None):
        positions, inv_freq, *versions = ctx.kept
        if versions != [positions._version, inv_freq._version]:
            raise RuntimeError("the positions or frequencies of a rotary call were changed in place before its "
                               "backward pass")
        interleaved, scale, inverse = ctx.how
        if dq is not None:
            dq, dk = _turn(dq, dk, positions, inv_freq, interleaved, scale, not inverse)
        elif dk is not None:
            dk = _turn(dk, None, positions, inv_freq, interleaved, scale, not inverse)[0]
        return dq, dk, None, None, None, None, None

    @staticmethod
    def jvp(ctx, dq, *rest):  # of q alone, as `_turn` calls it
        positions, inv_freq, *_ = ctx.kept
        return _Rotary.apply(dq, None, positions, inv_freq, *ctx.how)


def has_tangent(*xs: torch.Tensor | None) -> bool:
    """Whether forward-mode differentiation follows one of xs."""
    if forward_ad._current_level < 0:
        return False
    return any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in xs)


def _turn(q, k, positions, inv_freq, interleaved, scale, inverse):
    """(q, k) rotated, differentiably where gradients or tangents are asked for."""
    if has_tangent(q, k):  # a tensor at a time: one may have a tangent and the other not
        rest = positions, inv_freq, interleaved, scale, inverse
        return _Rotary.apply(q, None, *rest), None if k is None else _Rotary.apply(k, None, *rest)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _Rotary.apply(q, k, positions, inv_freq, interleaved, scale, inverse)
        return out if k is not None else (out, None)
    return _launch(q, k, positions, inv_freq, interleaved, scale, inverse)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
           interleaved: bool = False, attention_scaling: float = 1.0):
    """Rotate q [B, Hq, T, D] and k [B, Hkv, T, D] (or None) at `positions` ([T] or [B, T]) by
    the angles positions * inv_freq, in one kernel launch; returns (q_rot, k_rot), new tensors
    in the layout of the inputs (k_rot None without k).  Differentiable in q and k, in reverse and
    forward mode, and not in inv_freq (one that asks for gradients is refused).

    The first 2 * len(inv_freq) dims are rotated, the rest copied.  Pairs are (i, i + half), or
    (2i, 2i + 1) with `interleaved`.  Angles are formed in float64, the rotation in float32 with
    one rounding to the tensors' type (float32, bfloat16 or float16); cos and sin are multiplied
    by `attention_scaling`.  An inv_freq that is not float64 on the device is converted per call.
    Forward and backward can be captured into a CUDA graph, on torch's terms: no autograd graph
    of the same leaf tensors made outside the capture may be alive.
    """
    if (inv_freq.requires_grad and torch.is_grad_enabled()) or (forward_ad._current_level >= 0
                                                                  and has_tangent(inv_freq)):
        raise RuntimeError("rotary is not differentiable in its frequencies: detach inv_freq (apply_rope follows them)")
    return _turn(q, k, positions, inv_freq, interleaved, attention_scaling, False)
