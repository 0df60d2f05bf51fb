"""Global gradient norm and clipping coefficient in float64 (numpy)."""
from __future__ import annotations

import numpy as np


def norm(arrays, p: float) -> float:
    a = [np.abs(np.asarray(x, np.float64)).ravel() for x in arrays if np.size(x)]
    if not a:
        return 0.0
    if p == np.inf:
        return float(np.max([x.max() for x in a]))  # a NaN stays
    return float(sum((x ** p).sum() for x in a) ** (1.0 / p))


def coefficient(total: float, max_norm: float) -> float:
    c = np.float64(max_norm) / (np.float64(total) + 1e-6)
    return float(c if np.isnan(c) else min(c, 1.0))
