"""Tables of rotary positions: cosines and sines of position * frequency, computed in 64 bits and rounded once to fp32
(an fp32 angle of position 100000 is already off by 4e-3).  `ops.rotary` and `ops.fp8_kv_append` read them."""
import math
from typing import Optional

import torch


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_max: int = 8192, low: float = 1.0, high: float = 4.0, device=None):
    """(frequencies float64 [rot_dim / 2], factor on cosine and sine).  Pair i turns by base^(-2 i / rot_dim) per position;
    scaling stretches contexts by `factor`:

      None       as they are
      "linear"   every frequency / factor
      "ntk"      base * factor^(rot_dim / (rot_dim - 2)): the slowest pair is stretched by factor, the fastest not at all
      "yarn"     pairs that turn more than 32 times within original_max stay, fewer than once are / factor, a linear
                 ramp over the pairs between; cosine and sine times 0.1 ln(factor) + 1
      "banded"   pairs that turn more than `high` times within original_max stay, fewer than `low` times are / factor,
                 between them a blend that is linear in the number of turns
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and positive")
    if not factor > 0 or not base > 0:
        raise ValueError("factor and base must be positive")
    if scaling == "ntk":
        if rot_dim < 4:
            raise ValueError("ntk scaling needs rot_dim >= 4")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    index = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    freq = base ** (-index / rot_dim)
    if scaling in (None, "ntk"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if original_max < 1:
        raise ValueError("original_max must be positive")
    turns = original_max * freq / (2 * math.pi)
    if scaling == "yarn":
        if not base > 1:
            raise ValueError("yarn scaling needs base > 1")

        def pair_with(n):  # the (fractional) pair that turns n times within original_max
            return rot_dim * math.log(original_max / (n * 2 * math.pi)) / (2 * math.log(base))

        first, last = max(math.floor(pair_with(32.0)), 0), min(math.ceil(pair_with(1.0)), rot_dim - 1)
        if last <= 0:  # no pair turns even once: all of them are stretched
            ramp = torch.ones_like(freq)
        else:
            ramp = ((index / 2 - first) / max(last - first, 1e-3)).clamp(0, 1)
        return freq * (1 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    if scaling == "banded":
        if not high > low:
            raise ValueError("banded scaling needs high > low")
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return freq * keep + freq / factor * (1 - keep), 1.0
    raise ValueError(f"unknown scaling {scaling!r}")


def rotary_table(max_positions: int, rot_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_max: int = 8192, low: float = 1.0, high: float = 4.0, device=None) -> torch.Tensor:
    """float32 [max_positions, rot_dim]: per position rot_dim / 2 cosines, then rot_dim / 2 sines
    (see rotary_frequencies for the arguments)."""
    if max_positions < 1:
        raise ValueError("max_positions must be positive")
    freq, gain = rotary_frequencies(rot_dim, base, scaling, factor, original_max, low, high, device)
    table = torch.empty((max_positions, rot_dim), dtype=torch.float32, device=device)
    step = max(1, (1 << 24) // rot_dim)  # 64-bit angles of at most 128 MiB at a time
    for p in range(0, max_positions, step):
        angle = torch.arange(p, min(p + step, max_positions), dtype=torch.float64, device=device)[:, None] * freq
        table[p:p + step, : rot_dim // 2] = angle.cos() * gain
        table[p:p + step, rot_dim // 2 :] = angle.sin() * gain
    return table
