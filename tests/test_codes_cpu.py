"""CPU: the checks of the sampled-codes and lookup calls that need no GPU, and their 64-bit definitions themselves."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import codes_reference as ref
from vq_amd import Context, _lib


def bare():
    """A handle without a library context: everything here is refused before the library is called."""
    c = object.__new__(Context)
    c._h, c._L, c.device, c.K, c.D, c.M = None, None, 0, 3, 4, 0
    return c


def test_null_context_is_refused():
    L, bad = _lib.lib(), _lib.ERR_INVALID
    how = _lib.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None)
    need = C.c_size_t(0)
    assert L.vqhip_scores_device(None, None, 0, None, 0, None) == bad
    assert L.vqhip_sample_device(None, None, 0, 0, 1, 1, how, None, None, None, None) == bad
    assert L.vqhip_assign_sampled_workspace(None, 0, need) == bad
    assert L.vqhip_assign_sampled_device(None, None, 0, how, None, None, None, None, 0, None) == bad
    assert L.vqhip_lookup_device(None, None, 0, 1, 1, 1, None, 0, 1.0, None, 1, None) == bad
    assert L.vqhip_lookup_gradient_workspace(None, 0, 1, 1, need) == bad
    assert L.vqhip_lookup_gradient_device(None, None, 0, 1, None, 0, 1.0, 1, 1, None, 0, 1, 0, None, None, 0, None) == bad


def test_the_sampling_struct_is_the_header_s():
    assert C.sizeof(_lib.Sampling) == 48 and _lib.Sampling.top_k.offset == 12 and _lib.Sampling.dtemperature.offset == 16


def test_tensors_of_the_host_are_refused():
    c = bare()
    S, u, idx, T = torch.zeros(2, 5), torch.zeros(2), torch.zeros(2, dtype=torch.int32), torch.zeros(3, 4)
    for call in (lambda: c.scores(T), lambda: c.scores(T.numpy()), lambda: c.sample(S, u), lambda: c.sample(S.numpy(), u), lambda: c.sample(None, u),
                 lambda: c.assign_sampled(T, u), lambda: c.lookup(idx), lambda: c.lookup(idx.numpy()), lambda: c.lookup([0, 1]), lambda: c.lookup(idx, table=T),
                 lambda: c.lookup_gradient(T, idx), lambda: c.lookup_gradient(None, idx)):
        with pytest.raises((ValueError, AttributeError)):
            call()


def brute(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition once more, by sorting and cumulative sums."""
    l = np.where(np.isnan(row), -np.inf, np.asarray(row, np.float64))
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if not len(order):
        return 0, 0.0
    t, p, m = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    if t == 0 or p <= 0:
        return order[0], 1.0
    w = np.exp((l[order] - l[order[0]]) / t)
    n = len(order) if top_k == 0 else min(top_k, len(order))
    w = w[:n]
    before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
    keep = (before < p * w.sum()) | (np.arange(n) == 0) | (p >= 1)
    keep &= w >= m
    full = np.zeros(len(l))
    full[order[:n]] = np.where(keep, w, 0.0)
    c = np.cumsum(full)
    at = min(int(np.searchsorted(c, float(np.float32(u)) * c[-1], side="right")), len(l) - 1)
    return at, full[at] / c[-1]


def test_the_definition_of_a_draw():
    rng = np.random.default_rng(0)
    for trial in range(300):
        V = int(rng.integers(1, 60))
        row = rng.normal(size=V) * 3
        row[rng.random(V) < 0.2] = -np.inf
        row = np.round(row, 1) if trial % 3 == 0 else row
        how = dict(temperature=float(rng.choice([0.0, 0.5, 1.0, 3.0])), top_k=int(rng.choice([0, 1, 3, 20])), top_p=float(rng.choice([1.0, 0.9, 0.3, 0.0])),
                   min_p=float(rng.choice([0.0, 0.1])))
        u = float(np.float32(rng.random()))
        at, prob, margin = ref.sample_row(row, u, **how)
        if margin > 1e-9:
            assert (at, pytest.approx(prob, rel=1e-12)) == brute(row, u, **how)
    assert ref.sample_row([0.0, 0.0, 0.0, 0.0], 0.99, top_p=0.4)[0] == 1
    assert ref.sample_row([-math.inf, math.nan], 0.5)[:2] == (0, 0.0)
    assert ref.sample_row([1.0, math.inf, math.inf], 0.6)[:2] == (2, 0.5)


def test_the_definitions_of_scores_lookup_and_gradient():
    T, idx = np.arange(12.0).reshape(4, 3), np.array([[1, -1], [3, 4], [1, 0]])
    assert (ref.lookup(idx, T, 2.0)[0, 0] == [6, 8, 10]).all() and (ref.lookup(idx, T)[0, 1] == 0).all() and (ref.lookup(idx, T)[1, 1] == 0).all()
    G, n, size = ref.lookup_gradient(np.ones((3, 2, 3)) * -1.0, idx, 4, 0.5)
    assert n.tolist() == [1, 2, 0, 1] and (G[1] == -1).all() and (G[2] == 0).all() and (size[1] == 1).all()
    assert ref.scores([[1.0, 2.0]], [[1.0, 2.0], [4.0, 6.0]]).tolist() == [[0.0, -25.0]]
