"""Sampling a token per row from its definition, in float64, one row at a time."""
import numpy as np


def sample_row(logits, u, temperature, top_k=0, top_p=1.0, min_p=0.0) -> int:
    x = np.asarray(logits, dtype=np.float64)
    if np.isnan(x).any():
        return int(np.flatnonzero(np.isnan(x))[0])
    if not temperature > 0 or np.isneginf(x).all():
        return int(np.argmax(x))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if np.isposinf(top):
        w = np.isposinf(x[order]).astype(np.float64)
    else:
        w = np.where(np.isneginf(x[order]), 0.0,
                     np.exp(np.where(np.isneginf(x[order]), 0.0, x[order] - top)
                            / np.float64(temperature)))
    n = len(x)
    if 0 < top_k < n:
        n = int(top_k)
    if not top_p >= 1:
        cum = np.cumsum(w[:n])
        before = np.concatenate(([0.0], cum[:-1]))
        n = max(1, int((before < float(top_p) * cum[-1]).sum()))
    n = max(1, min(n, int(((w >= float(min_p)) & (w > 0)).sum())))
    cum = np.cumsum(w[:n])
    at = int((cum <= float(u) * cum[-1]).sum())
    return int(order[min(at, n - 1)])
