"""Sampled codes and codebook lookup in 64 bits, row by row from their definitions (include/vqhip.h): what the tests of
vqhip_scores_device, vqhip_sample_device, vqhip_lookup_device and vqhip_lookup_gradient_device compare with.  numpy only."""
import math

import numpy as np


def scores(X, W):
    X, W = np.asarray(X, np.float64), np.asarray(W, np.float64)
    return -np.stack([((X - w) ** 2).sum(1) for w in W], 1)


def sample_row(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> (idx, prob, margin): margin is how far u * Z lies from the nearest border of the draw, relative to Z, and how far
    top_p * Z1 lies from the nearest one of the nucleus (a test that reports a difference looks here first)."""
    temperature, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    l = [float("-inf") if math.isnan(v) else float(v) for v in row]
    alive = [j for j in range(len(l)) if l[j] > -math.inf]
    if not alive:
        return 0, 0.0, math.inf
    order = sorted(alive, key=lambda j: (-l[j], j))
    top = l[order[0]]
    if not (0.0 < temperature < math.inf) or top_p <= 0.0:
        return order[0], 1.0, math.inf
    w = {j: 1.0 if l[j] == top else math.exp((l[j] - top) / temperature) for j in alive}
    kept = order[:top_k] if top_k else order
    margin = math.inf
    if top_p < 1.0:
        border, mass, n = top_p * math.fsum(w[j] for j in kept), 0.0, 0
        sums = []
        for j in kept:
            sums.append(w[j])
            before = math.fsum(sums[:-1]) if len(kept) < 200 else mass
            if n and before >= border:
                break
            n += 1
            mass += w[j]
            margin = min(margin, abs(before - border) / border, abs(mass - border) / border)
        kept = kept[:n]
    kept = [j for j in kept if w[j] >= min(min_p, 1.0)]
    z = math.fsum(w[j] for j in kept)
    u = min(max(float(np.float32(u)), 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    at, mass = None, 0.0
    for j in sorted(kept):
        mass += w[j]
        if w[j] > 0.0:
            margin = min(margin, abs(mass - u * z) / z)
            if at is None or not done:
                at, done = j, mass > u * z
    return at, w[at] / z, margin


def lookup(idx, table, scale=1.0):
    table = np.asarray(table, np.float64)
    idx = np.asarray(idx, np.int64)
    out = np.zeros((*idx.shape, table.shape[1]))
    ok = (idx >= 0) & (idx < table.shape[0])
    out[ok] = table[idx[ok]] * float(np.float32(scale))
    return out


def lookup_gradient(grad, idx, K, scale=1.0):
    """-> (sums, counts, sums of absolute values: what the bound on a sum's rounding goes by)"""
    idx = np.asarray(idx, np.int64).reshape(-1)
    grad = np.asarray(grad, np.float64).reshape(idx.size, -1)
    ok = (idx >= 0) & (idx < K)
    sums, size = np.zeros((K, grad.shape[1])), np.zeros((K, grad.shape[1]))
    np.add.at(sums, idx[ok], grad[ok])
    np.add.at(size, idx[ok], np.abs(grad[ok]))
    s = float(np.float32(scale))
    return sums * s, np.bincount(idx[ok], minlength=K), size * abs(s)
