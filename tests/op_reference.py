"""64-bit plain implementations of the rotation, the paged append and the paged decode
attention, and bounds on how far a kernel's results may be from them.

Bounds.  u = torch.finfo(t).eps / 2 is the largest relative rounding error of type t.
Rotation: fp32 sine and cosine are within 2^-22 of exact (their argument rounded to fp32 after
an exact reduction, the functions' own 2 units, the scaling's rounding), products and sum
add 2^-23 of |x1| + |x2|; then one rounding to t.  Attention: every probability is rounded to t
once (u), scores carry the error of a D-term fp32 sum and of the exponential (2^-20), and the
output is rounded to t once."""

import torch


def u(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, positions, inv_freq, interleaved=False, scaling=1.0, sign=1):
    """x [B, H, T, D] in 64 bits, positions [B, T] or [T]."""
    x = x.detach().double()
    inv_freq = inv_freq.double().to(x.device)
    pos = (positions if positions.dim() == 2 else positions[None]).double()
    angle = sign * pos[:, None, :, None] * inv_freq
    c, s = angle.cos() * scaling, angle.sin() * scaling
    r = 2 * inv_freq.numel()
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    x1, x2 = x[..., first], x[..., second]
    y[..., first], y[..., second] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def rotate_bound(x, want, inv_freq, interleaved, scaling, dtype):
    """Elementwise bound on |got - want|."""
    x = x.detach().double().abs()
    r = 2 * inv_freq.numel()
    pair = torch.zeros_like(x)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    size = x[..., first] + x[..., second]
    pair[..., first], pair[..., second] = size, size
    fp32 = abs(scaling) * pair * (2.0 ** -22 + 2.0 ** -23)
    return fp32 + u(dtype) * (want.abs() + fp32) + torch.finfo(dtype).smallest_normal * u(dtype)


def gather(pages, table_row, n):
    """Rows [0, n) of one sequence, [Hkv, n, D] in 64 bits."""
    page = pages.shape[2]
    used = table_row[: -(-n // page)].long()
    return pages[used].transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n].double()


def attend(q, k_pages, v_pages, table, lens, scale, shared_len=0):
    """(out, bound) [B, 1, Hq, D] in 64 bits: decode attention over each sequence's rows, those
    below shared_len through table[0]."""
    b, hq, _, d = q.shape
    hkv, page = k_pages.shape[1], k_pages.shape[2]
    t = u(q.dtype)
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    ns = shared_len // page
    for i, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        row = torch.cat((table[0, :ns], table[i, ns:]))
        k, v = gather(k_pages, row, n), gather(v_pages, row, n)
        x = q[i, :, 0].double().reshape(hkv, hq // hkv, d)
        p = torch.softmax(x @ k.transpose(1, 2) * scale, dim=-1)
        out[i] = (p @ v).reshape(hq, d)
        size = (x.abs() @ k.abs().transpose(1, 2)).amax() * scale
        each = t + (d + 8) * 2.0 ** -23 * size + 2.0 ** -20
        # probabilities below the type's normal range lose up to half a smallest step each,
        # beside a sum of at least one
        tiny = n * torch.finfo(q.dtype).smallest_normal * t * v.abs().amax()
        absolute = (p @ v.abs()).reshape(hq, d)
        bound[i] = t * out[i].abs() + (1 + t) * (each * absolute + tiny)
    return out[:, None], bound[:, None]


def assert_bounded(got, want, bound, what=""):
    over = (got.double() - want).abs() - bound
    assert bool(torch.isfinite(got.double()).eq(torch.isfinite(want)).all()), f"{what}: finite where it should not be"
    worst = over.max().item()
    assert worst <= 0, (f"{what}: {worst:.3e} over the bound at {int(over.argmax())}, "
                        f"{int((over > 0).sum())} of {over.numel()} over")
