"""Rotary positions in 64 bits, straight from the definition, and the error bound of the kernels (shared by the tests)."""

import torch


def axis_of_frequency(half, sections, order):
    if not sections or len(sections) == 1:
        return [0] * half
    if order == "blocked":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = len(sections)
    axis = [0] * half
    for a in range(1, axes):
        for k in range(sections[a]):
            axis[a + axes * k] = a
    return axis


def rotate64(x, positions, inv_freq, sections=None, order="blocked", pairing="half", magnitude=1.0):
    """x [T, H, D], positions [T] or [A, T], inv_freq [R/2] (all on the CPU) -> float64."""
    half = inv_freq.numel()
    pos = positions.reshape(-1, x.shape[0]).double()
    angle = pos[axis_of_frequency(half, sections, order)].t() * inv_freq.double()  # [T, half]
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    y = x.double().clone()
    first = torch.arange(half)
    ia, ib = (first, first + half) if pairing == "half" else (2 * first, 2 * first + 1)
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def rotation_tolerance(x, ref, inv_freq, pairing, magnitude):
    """Largest error per element.  Sine and cosine: the fraction of a turn is rounded to fp32 (2^-25 turns = 1.9e-7 rad), the
    function adds at most 2 units of 2^-24 and the magnitude one rounding; each product and the sum round once more (2^-24
    relative each).  In all below 8e-7 of magnitude * (|a| + |b|).  Then one rounding to the output type: eps / 2 of the
    value, or half the smallest fp16 step near zero.  Elements past the rotated ones are copies."""
    half = inv_freq.numel()
    first = torch.arange(half)
    ia, ib = (first, first + half) if pairing == "half" else (2 * first, 2 * first + 1)
    size = torch.zeros_like(ref)
    both = x.double()[..., ia].abs() + x.double()[..., ib].abs()
    size[..., ia] = both
    size[..., ib] = both
    info = torch.finfo(x.dtype)
    tol = 8e-7 * abs(magnitude) * size
    return tol + torch.where(size > 0, info.eps / 2 * (ref.abs() + tol) + 2.0 ** -25, torch.zeros_like(ref))


def assert_rotated(out, x, positions, inv_freq, sections=None, order="blocked", pairing="half", magnitude=1.0):
    ref = rotate64(x, positions, inv_freq, sections, order, pairing, magnitude)
    tol = rotation_tolerance(x, ref, inv_freq, pairing, magnitude)
    excess = (out.cpu().double() - ref).abs() - tol
    assert excess.numel() == 0 or excess.max().item() <= 0, f"largest error past the bound: {excess.max().item():.3e}"
