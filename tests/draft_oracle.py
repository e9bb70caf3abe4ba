"""The verification of drafted tokens from its definition, in numpy's 64 bits: one request, one token after another."""
import numpy as np


def shares(row, temperature, top_k, top_p):
    """The probabilities that the sampler draws a row's token from, [vocab]; None for a row that has none."""
    row = np.asarray(row, dtype=np.float64)
    if np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any():
        return None
    order = np.lexsort((np.arange(row.size), -row))
    if temperature <= 0:
        order = order[:1]
        weights = np.ones(1)
    else:
        if top_k:
            order = order[:top_k]
        with np.errstate(over="ignore"):
            weights = np.exp((row[order] - row[order[0]]) / max(temperature, 1e-290))
        if top_p < 1:
            sums = np.cumsum(weights)
            count = int((sums < top_p * sums[-1]).sum()) + 1
            order, weights = order[:count], weights[:count]
    out = np.zeros(row.size)
    out[order] = weights / weights.sum()
    return out


def drawn(weights, uniform):
    """The first token at which the running sum exceeds its share of the total."""
    sums = np.cumsum(weights)
    over = np.nonzero(sums > uniform * sums[-1])[0]
    return int(over[0]) if over.size else int(np.nonzero(weights > 0)[0][-1])


def decide(target, drafts, uniforms, last, setting, draft=None):
    """(tokens, accepted) of one request: target [n + 1, vocab], drafts and uniforms [n], draft [n, vocab] or None;
    None where a row that matters cannot be used."""
    temperature, top_k, top_p = setting
    tokens = []
    for j in range(len(drafts) + 1):
        p = shares(target[j], *setting)
        q = None
        if j < len(drafts) and draft is not None and temperature > 0:
            q = shares(draft[j], *setting)
            if q is None:
                return None
        if p is None:
            return None
        if j == len(drafts):
            return tokens + [drawn(p, last)], j
        d = int(drafts[j])
        if uniforms[j] * (1.0 if q is None else q[d]) < p[d]:
            tokens.append(d)
            continue
        if temperature > 0:
            rest = p.copy()
            if q is None:
                rest[d] = 0.0
            else:
                rest = np.maximum(p - q, 0.0)
            if rest.sum() > 0:
                p = rest
        return tokens + [drawn(p, last)], j
