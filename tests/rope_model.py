"""The rotations of kc_rope from their formulas, in the host's widest type
(64-bit mantissas: a position of 2^31 leaves 2^-33 of the angle's unit)."""
import numpy as np

LD = np.longdouble
PI = LD("3.14159265358979323846264338327950288")


def frequencies(dim, base=10000.0, scaling="none", factor=1.0, original=0, low=0.0, high=0.0, freq_factors=None):
    i = np.arange(dim // 2).astype(LD)
    w = np.power(LD(np.float32(base)), -2 * i / dim)
    s, L = LD(np.float32(factor)), LD(original)
    low, high = LD(np.float32(low)), LD(np.float32(high))
    if freq_factors is not None:
        w = w / np.asarray(freq_factors, np.float32).astype(LD)
    if scaling == "linear":
        return w / s
    if scaling == "yarn":
        c = lambda x: dim * np.log(L / (2 * PI * x)) / (2 * np.log(LD(np.float32(base))))
        a, b = max(LD(0), np.floor(c(high))), min(LD(dim - 1), np.ceil(c(low)))
        r = np.clip((i - a) / max(LD("0.001"), b - a), 0, 1)
        return w * (r / s + 1 - r)
    if scaling == "bands":
        z = np.clip((L * w / (2 * PI) - low) / (high - low), 0, 1)
        return w * (z + (1 - z) / s)
    return w


def gain_of(scaling="none", factor=1.0, gain=0.0, **_):
    return LD(np.float32(gain)) if gain else 1 + LD("0.1") * np.log(LD(np.float32(factor))) if scaling == "yarn" else LD(1)


def turn(x, positions, dim, layout, gain=0.0, **how):
    """(result, magnitude): x [rows, heads, hd] turned, and |gain| (|a| + |b|) of
    each value's pair (its own size where nothing turns), for tolerances."""
    x = np.asarray(x).astype(LD)
    w, g = frequencies(dim, **how), gain_of(gain=gain, **how)
    angle = np.asarray(positions).astype(LD)[:, None] * w
    cos, sin = g * np.cos(angle)[:, None], g * np.sin(angle)[:, None]
    first = np.arange(dim // 2) if layout == "half" else np.arange(0, dim, 2)
    second = first + (dim // 2 if layout == "half" else 1)
    out, size = x.copy(), np.abs(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = abs(g) * (np.abs(a) + np.abs(b))
    return out, size
