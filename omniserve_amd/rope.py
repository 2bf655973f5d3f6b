"""Host-built RoPE coefficient tables for the KV4 kernels.

table[pos, i] = (cos, sin)(pos * scale / base**(2i/dim)) in float32, i < dim/2 -- the angle the
reference evaluates on the device (common/decoderMaskedMultiheadAttentionUtils.h:1147-1152).
Building it once on the host (numpy float32) makes the RoPE bit-reproducible and removes
powf/sincosf from the bandwidth-bound kernels.

`inverse_frequencies` is what the engine's layers use instead: they turn by position * frequency inside the kernel; it and `stretched_frequencies` are what
LmOps.rope and kv_store take, as a float64 tensor.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def inverse_frequencies(dims: int, base: float, scaling=None) -> list:
    """Rotation per position of the dims // 2 pairs (float64), base**(-2i/dims).

    scaling {factor, low, high, original}: frequencies of wavelengths below original / high stay, those above original / low are
    divided by factor, in between the two are blended linearly in original / wavelength."""
    out = []
    for i in range(dims // 2):
        f = float(base) ** (-2.0 * i / dims)
        if scaling:
            turns = scaling["original"] * f / (2.0 * math.pi)          # within the original context
            if turns < scaling["low"]:
                f /= scaling["factor"]
            elif turns <= scaling["high"]:
                s = (turns - scaling["low"]) / (scaling["high"] - scaling["low"])
                f = (1.0 - s) * f / scaling["factor"] + s * f
        out.append(f)
    return out


def stretched_frequencies(dims: int, base: float, factor: float, original: int, fast: float = 32.0, slow: float = 1.0):
    """Rotation per position of the dims // 2 pairs (float64) for a context `factor` times the original one, and what cosine and sine are multiplied with
    (YaRN, Peng et al. 2023): pairs that turn more than `fast` times within the original context keep their frequency, those that turn less than `slow`
    times are slowed down by factor, between them the two are blended linearly in the pair's number; scores are sharpened by (0.1 ln factor + 1)^2."""
    if dims < 2 or dims % 2 or not factor >= 1 or not fast > slow > 0:
        raise ValueError("an even number of dimensions, a factor of at least one and fast > slow > 0")
    pair = lambda turns: dims * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))      # noqa: E731
    first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dims - 1)
    out = []
    for i, f in enumerate(inverse_frequencies(dims, base)):
        keep = 1.0 - min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
        out.append(f * keep + f / factor * (1.0 - keep))
    return out, 0.1 * math.log(factor) + 1.0


_cache = {}
_retired = []     # superseded tables stay allocated: captured HIP graphs hold their raw pointers


def build_table_numpy(max_pos: int, dim: int, base: float, scale: float = 1.0) -> np.ndarray:
    half = dim // 2
    i = np.arange(half, dtype=np.float32)
    denom = np.power(np.float32(base), (np.float32(2.0) * i / np.float32(dim)).astype(np.float32)).astype(np.float32)
    t = (np.arange(max_pos, dtype=np.float32)[:, None] * np.float32(scale)).astype(np.float32)
    ang = (t / denom[None, :]).astype(np.float32)
    out = np.empty((max_pos, half, 2), np.float32)
    out[..., 0] = np.cos(ang)
    out[..., 1] = np.sin(ang)
    return out


def rope_table(max_pos: int, dim: int, base: float, scale: float, device) -> torch.Tensor:
    """Cached device table with at least `max_pos` rows (rounded up to a power of two >= 4096)."""
    key = (device, dim, base, scale)
    t = _cache.get(key)
    if t is None or t.shape[0] < max_pos:
        dim, base, scale = int(dim), float(base), float(scale)
        rows = 4096
        while rows < max_pos:
            rows *= 2
        if t is not None:
            _retired.append(t)
        t = torch.from_numpy(build_table_numpy(rows, dim, base, scale)).to(device)
        _cache[key] = t
    return t
