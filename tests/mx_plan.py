"""Which tile and how many splits the MXFP4 products take, estimated from their sizes as the library
does it, with the constants read from its sources."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parents[1] / "metal-marlin_amd" / "csrc"
CUS = 256
f = np.float32


def _costs(name: str) -> list[tuple]:
    text = (CSRC / name).read_text()
    rows = re.search(r"COSTS\[\] = \{(.*?)\};", text, re.S).group(1)
    return [tuple(float(v.rstrip("f")) for v in r.split(",")) for r in re.findall(r"\{([^{}]+)\}", rows)]


def _cdiv(a: int, b: int) -> int:
    return -(-a // b)


def _best(M, cols, stages, deep, most, costs, time):
    """(tile, splits) of the least time; `deep` stages at least for each of several splits."""
    best, least = None, None
    for t, c in enumerate(costs):
        tiles = _cdiv(M, int(c[0])) * _cdiv(cols, int(c[1]))
        for s in range(1, most + 1):
            if s > 1 and (tiles * s > 2 * CUS or stages < deep * s):
                break
            per = _cdiv(stages, s)
            splits = _cdiv(stages, per)
            us = time(tiles * splits, f(per), c)
            if splits > 1:
                us += f(2.5) + f(M) * f(cols) * f(4) * f(splits + 1) / f(3e6)
            if least is None or us < least:
                best, least = (t, splits), us
    return best


def product(M: int, N: int, K: int) -> tuple[int, int]:
    """Of the tiles 256 x 256, 128 x 256, 128 x 128, 64 x 128, 64 x 64; M > 64."""
    def time(blocks, per, c):
        return f(_cdiv(blocks, CUS)) * (per * f(c[2]) + f(c[3]))
    return _best(M, N, _cdiv(K, 256), 4, 8, _costs("mm_mx_gemm.hip"), time)


def gradient(M: int, N: int, K: int, fp32: bool) -> tuple[int, int]:
    """Of the tiles 128 x 256, 64 x 128, 32 x 128."""
    def time(blocks, per, c):
        rest = blocks % (2 * CUS)
        us = f(blocks // (2 * CUS)) * (per * f(c[3]) + f(c[4]))
        return us + (per * f(c[3] if rest > CUS else c[2]) + f(c[4]) if rest else f(0))
    return _best(M, K, _cdiv(N, 32 if fp32 else 64), 2, 16, _costs("mm_mx_backward.hip"), time)
