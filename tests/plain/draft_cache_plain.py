"""Plain forms in 64 bits of the operators of a cache that is drafted into and thinned out, request by request on the CPU."""
import math

import torch


def ancestors(parents):
    """Which nodes every node of a tree sees: itself and those above it, a truth value each."""
    n = len(parents)
    sees = torch.zeros((n, n), dtype=torch.bool)
    for i, up in enumerate(parents):
        if up >= 0:
            sees[i] = sees[up]
        sees[i, i] = True
    return sees


def attention(q, k, v, sees, scale):
    """q [n, Hq, hd], k and v [keys, Hkv, hd], sees [n, keys] -> out [n, Hq, hd] and the weights [Hq, n, keys]; a row that sees nothing
    has zeros in both, and what a row does not see is nothing to it, whatever stands there."""
    q, k, v = q.double(), k.double(), v.double()
    Hq, Hkv = q.shape[1], k.shape[1]
    out, weights = torch.zeros_like(q), torch.zeros((Hq, q.shape[0], k.shape[0]), dtype=torch.float64)
    if all(bool(x.isfinite().all()) for x in (q, k, v)):          # all rows at once
        kk, vv = (x.repeat_interleave(Hq // Hkv, 1).transpose(0, 1) for x in (k, v))
        x = torch.where(sees, q.transpose(0, 1) @ kk.transpose(1, 2) * scale, -math.inf)
        weights = torch.where(sees.any(1)[:, None], torch.softmax(x, -1), 0.0)
        return (weights @ vv).transpose(0, 1), weights
    for i in range(q.shape[0]):
        at = sees[i].nonzero()[:, 0]
        if at.numel() == 0:
            continue
        for h in range(Hq):
            x = k[at, h * Hkv // Hq] @ q[i, h] * scale
            p = torch.softmax(x, 0)
            weights[h, i, at] = p
            out[i, h] = p @ v[at, h * Hkv // Hq]
    return out, weights


def score_error(q, k, scale):
    """How far a score may be off, in units of e, when its products are summed in 32 bits: a rounding of half a step a sum, of the sum of
    the products' sizes (of finite ones)."""
    q, k = (x.double().nan_to_num(0.0, 0.0, 0.0) for x in (q, k))
    hd = q.shape[-1]
    g = q.shape[1] // k.shape[1]
    size = torch.einsum("nhd,khd->hnk", q.abs(), k.abs().repeat_interleave(g, 1)).max() if q.numel() and k.numel() else torch.tensor(0.0)
    return float((hd + 4) * 2.0 ** -24 * scale * size)


def commit(tokens, parents, targets, width):
    """The confirmed nodes of one tree and the token behind the last one."""
    if not tokens:
        return [], -1
    path = [0]
    while len(path) < width:
        last = path[-1]
        child = next((c for c in range(last + 1, len(tokens)) if parents[c] == last and tokens[c] == targets[last]), None)
        if child is None:
            break
        path.append(child)
    return path, targets[path[-1]]


def evict(mass, positions, end, budget, first, latest):
    """Of one request's places (lists): [(hole, filler)] of one kv head."""
    n = len(mass)
    if n <= budget:
        return []

    def worth(i):
        if positions[i] < first or positions[i] >= end - latest:
            return (2, 0.0)
        return (1, math.inf) if math.isnan(mass[i]) else (0, mass[i])

    order = sorted(range(n), key=lambda i: (-worth(i)[0], -worth(i)[1], i))
    stays = set(order[:budget])
    holes = [i for i in range(budget) if i not in stays]
    fillers = [i for i in range(budget, n) if i in stays]
    return list(zip(holes, fillers))
