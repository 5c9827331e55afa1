"""CPU oracle of what a layer does around the paged cache: rotary positions and
linear attention with a decay per head.

TEST INFRASTRUCTURE ONLY, as ``kv_oracle``.  ``rope`` fixes the fp32 operation
order that the GPU kernels implement (every place where it has to choose is
marked "CHOICE"); ``rope_f64`` and ``linear_attention`` are the definitions in
64 bits.
"""

from __future__ import annotations

import numpy as np

F32 = np.float32


def cos_sin_table(max_positions: int, rot: int, theta: float = 1e4) -> np.ndarray:
    """fp32 [max_positions, rot]: cos of the rot/2 pairs, then sin, from 64-bit angles."""
    inv = theta ** (-np.arange(0, rot, 2) / rot)
    angle = np.arange(max_positions)[:, None] * inv
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(F32)


def axis_of_pair(sections, interleaved: bool, half: int) -> np.ndarray:
    """The axis of each pair: runs of pairs, or (interleaved) the pairs a,
    a + A, a + 2A, .. of each axis a > 0, the others on axis 0."""
    if sections is None:
        return np.zeros(half, np.int64)
    n = len(sections)
    if not interleaved:
        return np.repeat(np.arange(n), sections)
    axis = np.zeros(half, np.int64)
    for a in range(1, n):
        axis[a:a + n * sections[a]:n][:sections[a]] = a
    return axis


def _pairs(rot: int, pairing: str):
    half = rot // 2
    if pairing == "half":
        return np.arange(half), np.arange(half) + half
    return np.arange(0, rot, 2), np.arange(1, rot, 2)


def _tables(positions, table, sections, interleaved):
    """cos, sin [T, rot/2] of each pair at its axis's position; NaN outside the table."""
    half = table.shape[1] // 2
    pos = np.asarray(positions, np.int64).reshape(-1, np.asarray(positions).shape[-1])
    at = pos[axis_of_pair(sections, interleaved, half)].T  # [T, half]
    inside = (at >= 0) & (at < table.shape[0])
    row = np.where(inside, at, 0)
    pair = np.arange(half)
    nan = table.dtype.type(np.nan)
    return np.where(inside, table[row, pair], nan), np.where(inside, table[row, half + pair], nan)


def rms_scale_f32(x: np.ndarray, eps: float) -> np.ndarray:
    """CHOICE: squares in fp32, added by a pairwise tree over neighbours, one
    multiply by 1/D, one add of eps, correctly rounded sqrt and reciprocal."""
    s = x * x
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    return F32(1) / np.sqrt(s * F32(1 / x.shape[-1]) + F32(eps))


def rope(x, positions, table, *, sections=None, interleaved=False, pairing="half", norm=None, eps=1e-6) -> np.ndarray:
    """Rotated (and first normalised) heads ``x`` [T, H, D] in fp32, not yet
    rounded to the output's type.

    CHOICE: x1 c - x2 s and x2 c + x1 s as two fp32 products and one fp32 add,
    each rounded by itself; the norm multiplies by the scale, then by the weight."""
    x = np.asarray(x).astype(F32)
    if norm is not None:
        x = x * rms_scale_f32(x, eps) * np.asarray(norm).astype(F32)
    c, s = (y[:, None, :] for y in _tables(positions, table, sections, interleaved))
    first, second = _pairs(table.shape[1], pairing)
    out = x.copy()
    a, b = x[..., first], x[..., second]
    with np.errstate(invalid="ignore", over="ignore"):
        out[..., first] = a * c - b * s
        out[..., second] = b * c + a * s
    return out


def rope_f64(x, positions, table, *, sections=None, interleaved=False, pairing="half", norm=None, eps=1e-6):
    """The same in 64 bits, pairs as complex numbers."""
    x = np.asarray(x).astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(norm).astype(np.float64)
    c, s = _tables(positions, table.astype(np.float64), sections, interleaved)
    first, second = _pairs(table.shape[1], pairing)
    out = x.copy()
    z = (x[..., first] + 1j * x[..., second]) * (c + 1j * s)[:, None, :]
    out[..., first], out[..., second] = z.real, z.imag
    return out


def linear_attention(q, k, v, log_decay, state, scale):
    """One sequence by its recurrence in 64 bits: q [n, H, D], k, v [n, Hkv, D],
    state [H, D, D]; returns (out [n, H, D], state)."""
    q, k, v = (np.asarray(x).astype(np.float64) for x in (q, k, v))
    group = q.shape[1] // k.shape[1]
    k, v = np.repeat(k, group, 1), np.repeat(v, group, 1)
    lam = np.exp(np.asarray(log_decay).astype(np.float64))[:, None, None]
    s = np.asarray(state).astype(np.float64)
    out = np.empty(q.shape)
    for t in range(q.shape[0]):
        s = s * lam + k[t, :, :, None] * v[t, :, None, :]
        out[t] = scale * np.einsum("hd,hde->he", q[t], s)
    return out, s
