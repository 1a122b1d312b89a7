"""8-bit rows, the norm in front of them and rotary positions, from their
definitions in include/trit_cuda.h, in numpy."""
import numpy as np


def rows_of(y):
    """8-bit rows of f32 rows y: (e4m3 numbers as f64, scales f32 [rows][groups]). The steps are f32, as defined."""
    y = np.asarray(y, np.float32)
    m, d = y.shape
    groups = (d + 127) // 128
    codes, scales = np.zeros((m, d)), np.ones((m, groups), np.float32)
    for b in range(groups):
        part = y[:, b * 128:b * 128 + 128]
        most = np.abs(part).max(1)
        scale = np.where(most > 0, np.maximum(most / np.float32(448), np.float32(2.0**-126)), np.float32(1)).astype(np.float32)
        v = (part * (np.float32(1) / scale)[:, None]).astype(np.float64)
        _, e = np.frexp(v)  # |v| in [2^(e-1), 2^e): 8 steps of 2^(e-4)
        step = np.exp2(np.maximum(e, -5).astype(np.float64) - 4)
        codes[:, b * 128:b * 128 + 128] = np.clip(np.rint(v / step) * step, -448, 448)
        scales[:, b] = scale
    return codes, scales


def values_of(codes, scales):
    """What 8-bit rows stand for, in 64 bits."""
    return codes * np.repeat(scales.astype(np.float64), 128, axis=1)[:, :codes.shape[1]]


def norm_f32(h, w, eps):
    """y = h f32(s w) in the defined f32 steps, s = f32(1 / sqrt(mean h^2 + eps)); where s is beyond 2^+-100, a power of two
    goes from s to h, so that s keeps its bits."""
    h = np.asarray(h, np.float32)
    s = 1.0 / np.sqrt((h.astype(np.float64)**2).mean(-1, keepdims=True) + eps)
    by = np.where((s < 2.0**-100) & (s > 0), 2.0**64, np.where(s > 2.0**100, 2.0**-64, 1.0))
    with np.errstate(invalid="ignore"):
        return h * (1 / by).astype(np.float32) * ((s * by).astype(np.float32) * np.asarray(w, np.float32)[None])


def turned(x, positions, frequencies, factor, interleaved):
    """x [m][heads][hd] with its first 2 len(frequencies) values turned, in 64 bits."""
    out = np.asarray(x, np.float64).copy()
    n = len(frequencies)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)[None]
    z = factor * np.exp(1j * angle)[:, None, :]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y = (out[..., a] + 1j * out[..., b]) * z
    out[..., a], out[..., b] = y.real, y.imag
    return out
