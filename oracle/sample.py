"""CPU restatement of spec::sample in 64 bits (numpy), from the definition in
include/npn_spec_verify.h: one row at a time, the ranks as a sorted list that the filters cut."""
import numpy as np

U_TOP = np.float64(1.0 - 2.0 ** -24)


def sample_row(logits, temperature, top_k, top_p, min_p, u):
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    top = x.max()
    if top == -np.inf:
        return -1
    if top == np.inf:
        x = np.where(x == np.inf, 0.0, -np.inf)
    ids = np.lexsort((np.arange(len(x)), -x))
    ids = ids[x[ids] > -np.inf]
    if not temperature > 0:
        return int(ids[0])
    with np.errstate(invalid="ignore"):
        w = np.exp((x[ids] - x[ids[0]]) / np.float64(temperature))
    if 0 < top_k < len(x):
        w = w[:top_k]
    keep = len(w)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = max(1, int((before < np.float64(top_p) * w.sum()).sum()))
    if min_p > 0:
        keep = min(keep, int((w >= min(np.float64(min_p), 1.0)).sum()))
    c = np.cumsum(w[:keep])
    goal = (0.0 if np.isnan(u) else min(max(np.float64(u), 0.0), U_TOP)) * c[-1]
    return int(ids[int((c <= goal).sum())])


def sample(logits, temperature, top_k, top_p, min_p, u):
    return np.array([sample_row(*row) for row in zip(logits, temperature, top_k, top_p, min_p, u)], np.int64)
