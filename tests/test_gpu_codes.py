"""vqhip_scores_device, vqhip_sample_device, vqhip_assign_sampled_device, vqhip_lookup_device and
vqhip_lookup_gradient_device against their definitions in 64 bits (tests/codes_reference.py).

Tolerances, derived before the first run (a rounding to f32 is off by at most 2^-24, to bf16 by 2^-8 ... relative):
  scores    (up to 16 values, or few prototypes; longer rows have a bound of their own below) every difference x - w rounds once (2^-24), its square and the running sum add a rounding per value: at most
            (D + 3) 2^-24 of the sum (all terms have one sign)
  sample    idx equal; prob one rounding of an f64 value: 2^-24, and 1e-9 for the f64 sums
  lookup    f32 product rounded once, then once to the type: 2^-24 (f32) or 2^-24 + eps/2
  gradient  a sum of n values in f32, in any order: at most n 2^-24 of the sum of the absolute values, the scaling 2^-24 more,
            then one rounding to the type, eps/2 of the value (and half the least subnormal)
"""
import ctypes as C

import numpy as np
import pytest
import torch

import codes_reference as ref
from vq_amd import Context, VqhipError, _lib

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def wide(t):
    return t.detach().double().cpu().numpy()


# ---------------------------------------------------------------------------------------------- scores
@pytest.mark.parametrize("N,D,K", [(150, 4, 3), (1, 1, 1), (7, 5, 2), (130, 16, 129), (257, 15, 300), (1000, 2, 1), (2, 16, 513), (300, 32, 11), (257, 17, 15), (600, 4, 32), (513, 3, 31),
                                   (515, 16, 32), (520, 7, 17), (1030, 9, 64), (259, 16, 40), (300, 5, 192)])
def test_scores(ctx, N, D, K):
    g = gen(N + D)
    W = torch.rand(K, D, generator=g) * 2 - 1
    X = W[torch.randint(K, (N,), generator=g)] + 0.1 * torch.randn(N, D, generator=g)
    X[0] = W[K - 1]
    ctx.set_prototypes(W.numpy())
    S = ctx.scores(X.cuda())
    want = ref.scores(X.numpy(), W.numpy())
    assert S.shape == (N, K) and S.dtype == torch.float32
    assert (np.abs(wide(S) - want) <= (D + 3) * 2.0 ** -24 * np.abs(want)).all()
    assert S[0, K - 1].item() == 0.0                         # direct form: a sample on a prototype is at distance 0


def test_scores_into_strided_rows_and_unaligned_inputs(ctx):
    g = gen(3)
    W, X = torch.randn(21, 13, generator=g), torch.randn(50, 13, generator=g)
    ctx.set_prototypes(W.numpy())
    buf = torch.full((50, 40), 7.0, device="cuda")
    x = torch.empty(50 * 13 + 1, device="cuda")[1:].view(50, 13).copy_(X)
    out = ctx.scores(x, out=buf[:, 3:24])
    want = ref.scores(X.numpy(), W.numpy())
    assert (np.abs(wide(out) - want) <= 16 * 2.0 ** -24 * np.abs(want)).all()
    assert (buf[:, :3] == 7).all() and (buf[:, 24:] == 7).all()
    assert torch.equal(ctx.scores(x), out.contiguous())


def test_scores_of_values_that_are_not_finite(ctx):
    W = torch.tensor([[0.0, 1.0], [2.0, 3.0]])
    ctx.set_prototypes(W.numpy())
    X = torch.tensor([[INF, 0.0], [NAN, 0.0], [1e30, 0.0], [0.0, 1.0]])
    S = ctx.scores(X.cuda()).cpu()
    assert (S[0] == -INF).all() and S[1].isnan().all() and (S[2] == -INF).all() and S[3].tolist() == [0.0, -8.0]


# ---------------------------------------------------------------------------------------------- sample
def check_sample(ctx, rows, u, dev=None, **how):
    """rows: cpu tensor N x V; how: numbers or cpu tensors."""
    dev = rows.cuda() if dev is None else dev
    on = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in how.items()}
    idx, prob = ctx.sample(dev, u.cuda(), **on)
    idx, prob = idx.cpu().numpy(), wide(prob)
    l = rows.float().numpy()
    for i in range(len(l)):
        one = {k: v[i].item() if isinstance(v, torch.Tensor) else v for k, v in how.items()}
        j, p, margin = ref.sample_row(l[i], u[i].item(), **one)
        if margin > 1e-12:
            assert idx[i] == j, (i, one, u[i].item(), idx[i], j, margin)
            assert abs(prob[i] - p) <= (2.0 ** -24 + 1e-9) * p, (i, prob[i], p)
    return idx, prob


HOWS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=50, temperature=1.3), dict(top_p=0.9), dict(top_p=0.05), dict(min_p=0.1),
        dict(top_k=40, top_p=0.95), dict(top_k=40, top_p=0.8, min_p=0.05, temperature=0.6), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0),
        dict(top_p=0.999), dict(temperature=100.0, top_p=0.5)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 256, 1000, 1025, 5000, 8193, 20001])
def test_sample(ctx, V, dtype):
    g = gen(V)
    N = 12 if V <= 1025 else 3
    for n, how in enumerate(HOWS):
        rows = (torch.randn(N, V, generator=g) * (0.1 + 4 * torch.rand(N, 1, generator=g))).to(TYPES[dtype])
        check_sample(ctx, rows, torch.rand(N, generator=g), **how)


@pytest.mark.parametrize("V", [3, 64, 300, 2000, 10000])
def test_sample_ties_and_masks(ctx, V):
    g = gen(V)
    flat = torch.zeros(V)
    few = torch.randint(0, 3, (V,), generator=g).float()
    masked = torch.randn(V, generator=g)
    masked[torch.rand(V, generator=g) < 0.5] = -INF
    low = torch.full((V,), torch.finfo(torch.float32).min)
    low_but_one = low.clone()
    low_but_one[V // 2] = 0.0
    one = torch.full((V,), -INF)
    one[V - 1] = -3.0
    nan = torch.randn(V, generator=g)
    nan[:: 2] = NAN
    zeros = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    two_inf = torch.randn(V, generator=g)
    two_inf[V // 3] = two_inf[V - 1] = INF
    rows = torch.stack([flat, few, masked, low, low_but_one, one, nan, zeros, two_inf, -flat - 1e30, torch.linspace(-88, 88, V)])
    for how in HOWS + [dict(top_k=V - 1 or 1), dict(top_k=V), dict(top_k=V + 7), dict(top_k=max(1, V // 2), top_p=0.5)]:
        for u in (0.0, 0.5, 0.999, 1.0 - 2.0 ** -24):
            check_sample(ctx, rows, torch.full((len(rows),), u), **how)


def test_sample_rows_with_nothing_to_draw(ctx):
    rows = torch.tensor([[-INF, -INF, -INF], [NAN, NAN, NAN], [NAN, -INF, 0.5], [-INF, 1.0, -INF]])
    for dtype in TYPES.values():
        for how in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.5), dict(temperature=0.0)):
            idx, prob = ctx.sample(rows.to(dtype).cuda(), torch.full((4,), 0.7, device="cuda"), **how)
            assert idx.tolist() == [0, 0, 2, 1] and prob.tolist() == [0.0, 0.0, 1.0, 1.0]


def test_sample_numbers_outside_the_unit_interval(ctx):
    rows = torch.zeros(6, 10).cuda()
    u = torch.tensor([-1.0, NAN, 1.0, 5.0, INF, -0.0]).cuda()
    idx, _ = ctx.sample(rows, u)
    assert idx.tolist() == [0, 0, 9, 9, 9, 0]


@pytest.mark.parametrize("V", [200, 3000, 9001])
def test_sample_parameters_per_row(ctx, V):
    g = gen(V + 1)
    N = 24
    rows = torch.randn(N, V, generator=g) * 3
    t = torch.rand(N, generator=g) * 2
    t[::5] = 0.0
    k = torch.randint(0, 100, (N,), generator=g).int()
    p = torch.rand(N, generator=g) * 1.2
    p = torch.where(p > 1, 1.0, p)
    m = torch.rand(N, generator=g) * 0.3
    check_sample(ctx, rows, torch.rand(N, generator=g), temperature=t, top_k=k, top_p=p, min_p=m)
    check_sample(ctx, rows, torch.rand(N, generator=g), temperature=t, top_p=0.9)
    check_sample(ctx, rows, torch.rand(N, generator=g), top_k=k, min_p=0.01)
    # what cannot be refused on the device is folded into the range
    idx, prob = ctx.sample(rows.cuda(), torch.zeros(N).cuda(), temperature=torch.tensor([NAN, -1.0, INF, 0.0] * 6).cuda())
    assert idx.tolist() == rows.argmax(1).tolist() and (prob == 1).all()
    a = ctx.sample(rows.cuda(), torch.full((N,), 0.4).cuda(), top_p=torch.tensor([NAN, 2.0, INF] * 8).cuda(), min_p=torch.tensor([NAN, -2.0, -INF] * 8).cuda(),
                   top_k=torch.tensor([0, -1, V] * 8).int().cuda())
    b = ctx.sample(rows.cuda(), torch.full((N,), 0.4).cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    idx, _ = ctx.sample(rows.cuda(), torch.full((N,), 0.4).cuda(), min_p=torch.full((N,), 7.0).cuda())
    assert idx.tolist() == rows.argmax(1).tolist()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sample_strided_rows(ctx, dtype):
    g = gen(9)
    buf = torch.full((9, 700), INF).to(TYPES[dtype])
    buf[:, 3:604] = torch.randn(9, 601, generator=g).to(TYPES[dtype])
    rows = buf[:, 3:604]
    check_sample(ctx, rows, torch.rand(9, generator=g), dev=buf.cuda()[:, 3:604], top_p=0.8)
    check_sample(ctx, rows[:1], torch.rand(1, generator=g), dev=buf.cuda()[:1, 3:604], top_k=7)


def test_sample_follows_the_distribution(ctx):
    """u on an even grid: how often an index comes up is its probability to within the grid (exactly one border each side)."""
    l = torch.tensor([1.0, -2.0, 0.5, 3.0, -INF, 0.0])
    n = 4096
    idx, prob = ctx.sample(l.repeat(n, 1).cuda(), (torch.arange(n) / n).cuda(), temperature=1.7, top_k=4)
    w = torch.exp(l.double() / 1.7)
    w[1] = w[4] = 0.0
    p = w / w.sum()
    share = torch.bincount(idx.long().cpu(), minlength=6) / n
    assert (share.double() - p).abs().max() <= 1.0 / n
    assert (torch.diff(idx.cpu()) >= 0).all()


# ---------------------------------------------------------------------------------------------- lookup
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,K,D", [(1, 1, 1), (5, 3, 4), (100, 7, 1), (33, 50, 128), (1000, 256, 128), (17, 11, 515), (64, 9, 4096), (3, 4, 12), (5000, 100, 66)])
def test_lookup(ctx, N, K, D, dtype):
    g = gen(N * D)
    table = torch.randn(K, D, generator=g).to(TYPES[dtype])
    idx = torch.randint(0, K, (N,), generator=g).int()
    idx[N // 2] = -1
    if N > 4:
        idx[3], idx[4] = K, 2 ** 31 - 1                       # outside: zero rows
    for scale in (1.0, -2.5, 11.313708):
        y = ctx.lookup(idx.cuda(), table=table.cuda(), scale=scale)
        want = ref.lookup(idx.numpy(), wide(table), scale)
        eps = 0.0 if dtype == "f32" else torch.finfo(TYPES[dtype]).eps / 2
        assert y.dtype == TYPES[dtype]
        tiny = torch.finfo(TYPES[dtype]).smallest_normal * (torch.finfo(TYPES[dtype]).eps / 2)
        assert (np.abs(wide(y) - want) <= (2.0 ** -24 + eps) * np.abs(want) + tiny).all()


def test_lookup_shapes_strides_and_prototypes(ctx):
    g = gen(2)
    W = torch.randn(10, 6, generator=g)
    ctx.set_prototypes(W.numpy())
    idx = torch.randint(-1, 10, (4, 5), generator=g).int()
    y = ctx.lookup(idx.cuda())
    want = torch.where((idx >= 0)[..., None], W[idx.long().clamp(min=0)], 0.0)
    assert torch.equal(y.cpu(), want)
    wide_table = torch.randn(10, 9, generator=g).half().cuda()
    buf = torch.full((20, 15), 5.0, device="cuda", dtype=torch.float16)
    out = ctx.lookup(idx.reshape(-1).cuda(), table=wide_table[:, 1:8], out=buf[:, 4:11])
    flat = idx.reshape(-1)
    want = torch.where((flat >= 0)[:, None], wide_table.cpu()[flat.long().clamp(min=0)][:, 1:8], torch.tensor(0.0).half())
    assert torch.equal(out.cpu(), want) and (buf[:, :4] == 5).all() and (buf[:, 11:] == 5).all()
    assert ctx.lookup(torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 6)


# ---------------------------------------------------------------------------------------------- gradient
def check_gradient(ctx, grad, idx, K, scale=1.0, out_dtype=torch.float32, dev=None):
    D = grad.shape[-1]
    G, counts = ctx.lookup_gradient(grad.cuda() if dev is None else dev, idx.cuda(), K=K, scale=scale, out_dtype=out_dtype, want_counts=True)
    want, n, size = ref.lookup_gradient(wide(grad), idx.numpy(), K, scale)
    assert G.shape == (K, D) and G.dtype == out_dtype and counts.dtype == torch.int32
    assert (counts.cpu().numpy() == n).all()
    eps = 0.0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2
    tiny = torch.finfo(out_dtype).smallest_normal * (torch.finfo(out_dtype).eps / 2)
    bound = (n[:, None] + 1) * 2.0 ** -24 * size
    assert (np.abs(wide(G) - want) <= bound + eps * (np.abs(want) + bound) + tiny).all()
    return G, counts


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,K,D", [(1, 1, 1), (2, 5, 3), (150, 3, 4), (9, 200, 64), (1000, 256, 128), (8191, 17, 5), (8192, 1000, 8), (8193, 1000, 8),
                                   (20000, 2047, 16), (20000, 2048, 16), (30000, 100000, 4), (600, 33, 515), (100, 50, 1030), (70001, 2, 2)])
def test_gradient(ctx, N, K, D, dtype):
    g = gen(N + K + D)
    grad = torch.randn(N, D, generator=g).to(TYPES[dtype])
    idx = (torch.rand(N, generator=g) ** 3 * (K + 1)).int() - 1          # skewed, some -1
    check_gradient(ctx, grad, idx, K)
    if dtype != "f32":
        check_gradient(ctx, grad, idx, K, scale=0.25, out_dtype=TYPES[dtype])


@pytest.mark.parametrize("N", [5, 4096, 30000])
def test_gradient_of_one_crowded_index_and_of_none(ctx, N):
    g = gen(N)
    grad = torch.randn(N, 24, generator=g)
    check_gradient(ctx, grad, torch.full((N,), 3, dtype=torch.int32), 5, scale=-1.5)
    check_gradient(ctx, grad, torch.full((N,), -1, dtype=torch.int32), 5)
    check_gradient(ctx, grad, torch.full((N,), 4, dtype=torch.int32), 5)
    idx = torch.full((N,), 2, dtype=torch.int32)
    idx[::7] = -1
    idx[-1] = 0
    check_gradient(ctx, grad, idx, 5)


def test_gradient_does_not_read_padded_rows(ctx):
    grad = torch.ones(50, 6)
    idx = (torch.arange(50) % 4).int()
    idx[::3] = -1
    grad[::3] = NAN
    G, _ = ctx.lookup_gradient(grad.cuda(), idx.cuda(), K=4, want_counts=True)
    assert torch.isfinite(G).all() and G.sum().item() == 6 * (idx >= 0).sum().item()


@pytest.mark.parametrize("out_dtype", ["f32", "bf16"])
def test_gradient_accumulates_and_writes_strided_rows(ctx, out_dtype):
    g = gen(5)
    t = TYPES[out_dtype]
    grad = torch.randn(300, 10, generator=g).bfloat16()
    idx = torch.randint(0, 12, (300,), generator=g).int()
    idx[idx == 7] = 8                                                    # row 7 stays unnamed
    before = torch.randn(12, 20, generator=g).to(t)
    buf = before.clone().cuda()
    out = ctx.lookup_gradient(grad.cuda(), idx.cuda(), K=12, scale=0.5, out=buf[:, 5:15], accumulate=True)
    want, n, size = ref.lookup_gradient(wide(grad), idx.numpy(), 12, 0.5)
    want = want + wide(before)[:, 5:15]
    eps = 0.0 if out_dtype == "f32" else 2.0 ** -8
    bound = (n[:, None] + 2) * 2.0 ** -24 * (size + np.abs(wide(before)[:, 5:15]))
    assert (np.abs(wide(out) - want) <= bound + eps * (np.abs(want) + bound)).all()
    assert torch.equal(buf[7].cpu(), before[7])
    assert torch.equal(buf[:, :5].cpu(), before[:, :5]) and torch.equal(buf[:, 15:].cpu(), before[:, 15:])


def test_gradient_is_that_of_the_lookup(ctx):
    """d/dT of sum(c * lookup(T)) by differences: the lookup is linear in T, so a step of any size is exact up to rounding."""
    g = gen(11)
    T, c = torch.randn(6, 5, generator=g), torch.randn(40, 5, generator=g)
    idx = torch.randint(-1, 6, (40,), generator=g).int()
    G = wide(ctx.lookup_gradient(c.cuda(), idx.cuda(), K=6, scale=1.5))
    f = lambda t: (wide(ctx.lookup(idx.cuda(), table=t.cuda(), scale=1.5)) * wide(c)).sum()
    for k in range(6):
        for d in range(5):
            up, down = T.clone(), T.clone()
            up[k, d] += 1.0
            down[k, d] -= 1.0
            step = (up[k, d].double() - down[k, d].double()).item()
            # each of the 40 looked-up values is rounded to f32 (they stay below 8 in size): 40 * 8 * 1.5 * 2^-24 * |c| on each side
            assert abs((f(up) - f(down)) / step - G[k, d]) <= 40 * 12 * 4 * 2.0 ** -24


def test_gradient_strided_rows_and_shapes(ctx):
    g = gen(6)
    buf = torch.randn(90, 37, generator=g).half()
    idx = torch.randint(0, 20, (90,), generator=g).int()
    check_gradient(ctx, buf[:, 2:33], idx, 20, dev=buf.cuda()[:, 2:33], out_dtype=torch.float16)
    a = ctx.lookup_gradient(buf.cuda().view(9, 10, 37), idx.cuda().view(9, 10), K=20)
    assert torch.equal(a, ctx.lookup_gradient(buf.cuda(), idx.cuda(), K=20))
    G, n = ctx.lookup_gradient(torch.empty(0, 4, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), K=3, want_counts=True)
    assert (G == 0).all() and G.shape == (3, 4) and n.tolist() == [0, 0, 0]
    keep = torch.ones(3, 4, device="cuda")
    ctx.lookup_gradient(torch.empty(0, 4, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), K=3, out=keep, accumulate=True)
    assert (keep == 1).all()


@pytest.mark.parametrize("N,K,D", [(5000, 40, 32), (50000, 300, 12), (20000, 3, 256)])
def test_gradient_has_the_same_bits_every_time(ctx, N, K, D):
    g = gen(N)
    grad, idx = torch.randn(N, D, generator=g).cuda(), torch.randint(0, K, (N,), generator=g).int().cuda()
    first = ctx.lookup_gradient(grad, idx, K=K)
    for _ in range(3):
        assert torch.equal(ctx.lookup_gradient(grad, idx, K=K), first)


# ---------------------------------------------------------------------------------------------- together
def test_sampled_codes_train_a_codebook(ctx):
    """The run a program makes: draw a code per sample, decode it, bring the gradient of the decoding back to the codebook, and
    take the step (W moves towards the samples that drew each code)."""
    g = gen(21)
    W = torch.randn(64, 32, generator=g)
    X = (W[torch.randint(64, (3000,), generator=g)] + 0.2 * torch.randn(3000, 32, generator=g)).cuda()
    u = torch.rand(3000, generator=g).cuda()
    ctx.set_prototypes(W.numpy())
    idx, prob = ctx.assign_sampled(X, u, temperature=4.0, top_k=8, top_p=0.99)
    S = ctx.scores(X)
    a, b = ctx.sample(S, u, temperature=4.0, top_k=8, top_p=0.99)
    assert torch.equal(a, idx) and torch.equal(b, prob)
    nearest = ctx.assign(X)[0]
    greedy, _ = ctx.assign_sampled(X, u, temperature=0.0)
    best = S.gather(1, nearest.long()[:, None]) - S.gather(1, greedy.long()[:, None])
    assert best.abs().max() <= 64 * 2.0 ** -24 * S.abs().max()          # ties of f32 aside, temperature 0 is assign
    Y = ctx.lookup(idx)
    assert torch.equal(Y.cpu(), W[idx.long().cpu()])
    dY = 2 * (Y - X)
    G, n = ctx.lookup_gradient(dY, idx, want_counts=True)
    want, counts, size = ref.lookup_gradient(wide(dY), idx.cpu().numpy(), 64)
    assert (n.cpu().numpy() == counts).all() and (np.abs(wide(G) - want) <= (counts[:, None] + 1) * 2.0 ** -24 * size).all()
    sums = ctx.lookup_gradient(X, idx)
    means = torch.where(n[:, None] > 0, sums / n.clamp(min=1)[:, None], torch.from_numpy(W.numpy()).cuda())
    moved = torch.where(n[:, None] > 0, W.cuda() - G / (2 * n.clamp(min=1)[:, None]), W.cuda())
    assert (means - moved).abs().max() <= 1e-4                            # the full step of the batch update lands on the means


def test_assign_sampled_in_small_workspaces(ctx):
    g = gen(22)
    W, X, u = torch.randn(10, 4, generator=g), torch.randn(101, 4, generator=g).cuda(), torch.rand(101, generator=g).cuda()
    ctx.set_prototypes(W.numpy())
    t = (torch.rand(101, generator=g) + 0.5).cuda()
    idx, prob = ctx.assign_sampled(X, u, temperature=t)
    L = _lib.lib()
    for rows in (1, 7, 100, 101):
        work, i2, p2 = torch.empty(rows * 10, device="cuda"), torch.empty_like(idx), torch.empty_like(prob)
        how = _lib.Sampling(1.0, 1.0, 0.0, 0, t.data_ptr(), None, None, None)
        rc = L.vqhip_assign_sampled_device(ctx._h, X.data_ptr(), 101, how, u.data_ptr(), i2.data_ptr(), p2.data_ptr(), work.data_ptr(), rows * 40,
                                           torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(i2, idx) and torch.equal(p2, prob)


def test_on_another_stream_and_in_a_graph(ctx):
    g = gen(23)
    W = torch.randn(32, 16, generator=g)
    ctx.set_prototypes(W.numpy())
    X, u = torch.randn(9000, 16, generator=g).cuda(), torch.rand(9000, generator=g).cuda()

    def step():
        idx, prob = ctx.assign_sampled(X, u, temperature=3.0, top_p=0.9)
        Y = ctx.lookup(idx, scale=2.0)
        G, n = ctx.lookup_gradient(Y, idx, want_counts=True)
        return idx, prob, Y, G, n

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(second):
        held2 = step()
    for turn in range(4):
        X.copy_(torch.randn(9000, 16, generator=g))
        u.copy_(torch.rand(9000, generator=g))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), turn
        with torch.cuda.stream(side):
            second.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held2)) and all(torch.equal(a, b) for a, b in zip(want, held)), turn
        assert torch.equal(step()[3], want[3])


# ---------------------------------------------------------------------------------------------- refusals
def test_refusals(ctx):
    W = torch.randn(5, 4)
    ctx.set_prototypes(W.numpy())
    X, u, idx = torch.randn(3, 4).cuda(), torch.rand(3).cuda(), torch.zeros(3, dtype=torch.int32).cuda()
    S = ctx.scores(X)
    for bad in (X.double(), X.cpu(), X.t(), X[:, :3]):
        with pytest.raises(ValueError):
            ctx.scores(bad)
    with pytest.raises(ValueError):
        ctx.scores(X, out=torch.empty(3, 6, device="cuda"))
    for bad in (S.double(), S.cpu(), S[0], S.t(), S[:, ::2], S[:1].expand(3, 5)):
        with pytest.raises(ValueError):
            ctx.sample(bad, u)
    for bad in (u.double(), u[:2], u.cpu(), 0.5, None):
        with pytest.raises(ValueError):
            ctx.sample(S, bad)
    for how in (dict(temperature=-1.0), dict(temperature=NAN), dict(temperature=INF), dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=NAN), dict(min_p=2.0),
                dict(min_p=NAN)):
        with pytest.raises(VqhipError) as e:
            ctx.sample(S, u, **how)
        assert e.value.code == _lib.ERR_INVALID
        with pytest.raises(VqhipError):
            ctx.assign_sampled(X, u, **how)
    for how in (dict(top_k=-1), dict(top_k=1 << 32), dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:2]), dict(min_p=u.cpu())):
        with pytest.raises(ValueError):
            ctx.sample(S, u, **how)
    with pytest.raises(VqhipError):
        ctx.sample(torch.empty(3, 0, device="cuda"), u)
    for bad in (idx.long(), idx.cpu(), torch.zeros(6, dtype=torch.int32).cuda()[::2]):
        with pytest.raises(ValueError):
            ctx.lookup(bad)
        with pytest.raises(ValueError):
            ctx.lookup_gradient(X, bad)
    with pytest.raises(ValueError):
        ctx.lookup(idx, table=X.double())
    with pytest.raises(ValueError):
        ctx.lookup(idx, table=X, out=torch.empty(3, 4, dtype=torch.float16, device="cuda"))
    for bad in (X[:2], X.double(), X[:1].expand(3, 4), X.t()):
        with pytest.raises(ValueError):
            ctx.lookup_gradient(bad, idx)
    with pytest.raises(ValueError):
        ctx.lookup_gradient(X, idx, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        ctx.lookup_gradient(X, idx, accumulate=True)
    with pytest.raises(ValueError):
        ctx.lookup_gradient(X, idx, K=0)
    with pytest.raises(ValueError):
        ctx.lookup_gradient(X, idx, out=torch.empty(4, 4, device="cuda"))
    ctx.set_omega(np.eye(4, dtype=np.float32))
    for call in (lambda: ctx.scores(X), lambda: ctx.assign_sampled(X, u)):
        with pytest.raises(VqhipError) as e:
            call()
        assert e.value.code == _lib.ERR_UNSUPPORTED
    ctx.set_omega(None)
    fresh = Context(0)
    for call in (lambda: fresh.scores(torch.empty(3, 0, device="cuda")), lambda: fresh.lookup(idx)):
        with pytest.raises(VqhipError) as e:
            call()
        assert e.value.code == _lib.ERR_STATE
    fresh.close()


def test_c_refusals(ctx):
    """What the handle above never passes: the C entry points' own checks."""
    ctx.set_prototypes(np.zeros((5, 4), np.float32))
    L, h = _lib.lib(), ctx._h
    b = torch.zeros(4096, device="cuda")
    p = b.data_ptr()
    how = _lib.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None)
    bad = _lib.ERR_INVALID
    assert L.vqhip_scores_device(None, p, 1, p, 5, None) == bad
    assert L.vqhip_scores_device(h, None, 1, p, 5, None) == bad and L.vqhip_scores_device(h, p, 1, None, 5, None) == bad
    assert L.vqhip_scores_device(h, p, 1, p, 4, None) == bad and L.vqhip_scores_device(h, p + 2, 1, p, 5, None) == bad
    assert L.vqhip_scores_device(h, p, 1 << 62, p, 5, None) == bad
    assert L.vqhip_sample_device(h, p, 0, 1, 5, 5, None, p, p, p, None) == bad
    for args in ((None, 0, 1, 5, 5, how, p, p, p), (p, 3, 1, 5, 5, how, p, p, p), (p, 0, 1, 0, 5, how, p, p, p), (p, 0, 1, 5, 4, how, p, p, p),
                 (p, 0, 1, 1 << 31, 1 << 31, how, p, p, p), (p, 0, 1, 5, 5, how, None, p, p), (p, 0, 1, 5, 5, how, p, None, p), (p + 2, 0, 1, 5, 5, how, p, p, p),
                 (p, 0, 1, 5, 5, how, p + 1, p, p), (p, 0, 1 << 62, 5, 5, how, p, p, p)):
        assert L.vqhip_sample_device(h, *args, None) == bad
    assert L.vqhip_assign_sampled_device(h, p, 1, how, p, p, p, p, 19, None) == bad
    assert L.vqhip_assign_sampled_device(h, p, 1, how, p, p, p, None, 20, None) == bad
    assert L.vqhip_assign_sampled_workspace(h, 1, None) == bad
    for args in ((p, 5, 5, 4, 4, p, 1, 1.0, p, 4), (p, 0, 0, 4, 4, p, 1, 1.0, p, 4), (p, 0, 5, 0, 4, p, 1, 1.0, p, 4), (p, 0, 5, 4, 3, p, 1, 1.0, p, 4),
                 (p, 0, 5, 4, 4, None, 1, 1.0, p, 4), (p, 0, 5, 4, 4, p, 1, 1.0, None, 4), (p, 0, 5, 4, 4, p, 1, 1.0, p, 3), (None, 1, 5, 4, 4, p, 1, 1.0, p, 4),
                 (None, 0, 6, 4, 4, p, 1, 1.0, p, 4), (p + 2, 0, 5, 4, 4, p, 1, 1.0, p, 4), (p, 0, 5, 4, 4, p + 2, 1, 1.0, p, 4)):
        assert L.vqhip_lookup_device(h, *args, None) == bad, args
    need = C.c_size_t(0)
    assert L.vqhip_lookup_gradient_workspace(h, 10, 5, 4, C.byref(need)) == 0 and need.value > 0
    assert L.vqhip_lookup_gradient_workspace(h, 1 << 31, 5, 4, C.byref(need)) == bad
    w = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    q, n = w.data_ptr(), w.numel()
    ok = dict(dY=p, dtype=0, ldy=4, idx=p, N=3, scale=1.0, K=5, D=4, dT=p + 8192, out=0, ldt=4, acc=0, counts=None, work=q, bytes=n, stream=None)
    for change in (dict(dtype=7), dict(out=1), dict(ldy=3), dict(ldt=3), dict(work=q + 8), dict(bytes=16), dict(work=None), dict(dT=None), dict(dY=None),
                   dict(idx=None), dict(K=0), dict(D=0), dict(N=1 << 31), dict(counts=p + 1), dict(dY=p + 2), dict(K=1 << 31)):
        assert L.vqhip_lookup_gradient_device(h, *{**ok, **change}.values()) == bad, change
    assert L.vqhip_lookup_gradient_device(h, *ok.values()) == 0
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------- scores on the matrix cores
@pytest.mark.parametrize("N,D,K", [(257, 17, 300), (2, 32, 513), (129, 32, 16), (70, 17, 64), (1, 33, 1), (64, 128, 256), (33, 784, 100), (129, 255, 127), (2, 1000, 513), (130, 64, 129), (65, 100, 70), (300, 128, 256), (20, 785, 33), (4100, 40, 2100), (2048, 36, 4096)])
@pytest.mark.parametrize("offset", [0.0, 100.0])
def test_scores_in_the_expanded_form(ctx, N, D, K, offset):
    """Rows of more than 16 values (but for a few prototypes): distances not below 1/16 of B = |x - c|^2 + |w - c|^2 come from B - 2 (x - c).(w - c).  Its
    roundings, with e = 2^-24: each centred value 1 e of itself, which moves the distance by at most 2 sqrt(dist) e (|x - c| + |w - c|)
    <= 4 e B; each norm a sum of D squares, D e of itself, together D e B; the product a chain of D terms whose absolute
    values sum to at most B / 2, doubled D e B; the two last additions 2 e B.  (2 D + 6) e B <= 16 (2 D + 6) e dist;
    the tests hold it to half of that."""
    g = gen(N + D)
    W = torch.rand(K, D, generator=g) * 2 - 1 + offset
    X = W[torch.randint(K, (N,), generator=g)] + 0.1 * torch.randn(N, D, generator=g)
    X[:: 3] = torch.rand(len(X[:: 3]), D, generator=g) * 4 - 2 + offset
    X[0] = W[K - 1]
    ctx.set_prototypes(W.numpy())
    S = wide(ctx.scores(X.cuda()))
    want = -torch.cdist(X.double(), W.double(), compute_mode="donot_use_mm_for_euclid_dist").square().numpy()
    assert (np.abs(S - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want) + 1e-300).all()
    assert S[0, K - 1] == 0.0


@pytest.mark.parametrize("N", [70, 9000])
@pytest.mark.parametrize("crowd", [1, 2, 64])
def test_scores_of_crowded_prototypes(ctx, N, crowd):
    """Prototypes in `crowd` tight groups, a group's samples among them: from a few close pairs a tile to nothing else.  Close
    pairs are measured in the direct form: (D + 3) e of the distance; the others as above."""
    D, K = 48, 900
    g = gen(crowd)
    centre = torch.randn(crowd, D, generator=g)
    W = centre[torch.arange(K) % crowd] + 1e-3 * torch.randn(K, D, generator=g)
    X = centre[torch.randint(crowd, (N,), generator=g)] + 1e-3 * torch.randn(N, D, generator=g)
    ctx.set_prototypes(W.numpy())
    buf = torch.full((N, K + 5), 3.0, device="cuda")
    S = wide(ctx.scores(X.cuda(), out=buf[:, 2:K + 2]))
    want = -torch.cdist(X.double(), W.double(), compute_mode="donot_use_mm_for_euclid_dist").square().numpy()
    assert (np.abs(S - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)).all()
    assert (buf[:, :2] == 3).all() and (buf[:, K + 2:] == 3).all()


def test_scores_of_long_rows_that_are_not_finite(ctx):
    W = torch.randn(70, 40)
    W[3, 5], W[4, 6], W[5, 7] = INF, NAN, 3e38
    X = torch.randn(80, 40)
    X[0, 0], X[1, 1], X[2, 2], X[3, 5] = INF, NAN, 1e30, INF
    ctx.set_prototypes(W.numpy())
    S = wide(ctx.scores(X.cuda()))
    with np.errstate(over="ignore", invalid="ignore"):
        d = (X.numpy()[:, None, :] - W.numpy()[None]).astype(np.float32)
        want = -(d * d).sum(2).astype(np.float64)
    bad = ~np.isfinite(want)
    assert (np.isnan(S) == np.isnan(want)).all() and (S[bad & ~np.isnan(want)] == want[bad & ~np.isnan(want)]).all()
    assert np.isfinite(S[~bad]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [5, 250, 1001, 1030, 9001])
def test_sample_rows_that_begin_anywhere(ctx, V, dtype):
    """Rows at every offset from a 16-byte boundary; what lies beside them would win if it were read."""
    g = gen(V)
    t = TYPES[dtype]
    buf = torch.full((17, V + 9), 3e4).to(t)
    for off in range(9):
        rows = (torch.randn(17, V, generator=g) * 3).to(t)
        whole = buf.clone()
        whole[:, off:off + V] = rows
        u = torch.rand(17, generator=g)
        check_sample(ctx, rows, u, dev=whole.cuda()[:, off:off + V], **[dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0)][off % 5])
    first = torch.full((3, V), 0.0).to(t)
    first[0, 0] = first[1, V - 1] = 50.0
    first[2, V // 2] = 50.0
    idx, _ = ctx.sample(first.cuda(), torch.full((3,), 0.5).cuda(), top_p=0.5)
    assert idx.tolist() == [0, V - 1, V // 2]


@pytest.mark.parametrize("N,K,D", [(1, 70000, 3), (64, 64, 64), (1024, 1, 512), (1025, 4096, 24), (4096, 3, 40), (4096, 40000, 96), (4097, 40000, 96), (3001, 997, 515),
                                   (700, 65, 9000), (4000, 9, 4096), (300, 3000, 3000)])
@pytest.mark.parametrize("spread", ["even", "one", "few"])
def test_gradient_on_both_sides_of_one_launch(ctx, N, K, D, spread):
    """Sizes around the rule for the form that is one launch, with even, single and crowded indices; sums and counts, and a second
    call that adds to the first's."""
    g = gen(N + K)
    grad = torch.randn(N, D, generator=g)
    idx = torch.randint(-1, K, (N,), generator=g).int()
    if spread == "one":
        idx[:] = K // 2
    if spread == "few":
        idx = torch.where(torch.rand(N, generator=g) < 0.9, torch.minimum(idx, torch.tensor(2).int()), idx)
    G, _ = check_gradient(ctx, grad, idx, K, scale=2.0)
    out = ctx.lookup_gradient(grad.cuda(), idx.cuda(), K=K, scale=2.0, out=G.clone(), accumulate=True)
    assert torch.equal(out, 2 * G)                                   # x + x is exact


# ---------------------------------------------------------------------------------------------- what the calls allow at their ends
@pytest.mark.parametrize("V", [1500, 9001, 40000])
@pytest.mark.parametrize("order", ["up", "down", "block", "few values"])
def test_sample_rows_in_order(ctx, V, order):
    """The largest scores side by side, so that one wave's part of the row holds all of them, and long runs of equal ones."""
    g = gen(V)
    row = torch.randn(V, generator=g) * 3
    if order != "few values":
        row = row.sort(descending=order == "down").values
    if order == "block":
        row = row.roll(V // 3)
    if order == "few values":
        row = torch.randint(0, 5, (V,), generator=g).float()
    rows = row.repeat(4, 1)
    u = torch.tensor([0.01, 0.4, 0.77, 0.999])
    for how in (dict(top_k=100), dict(top_k=129), dict(top_k=256), dict(top_k=257), dict(top_k=700, top_p=0.9), dict(top_p=0.95), dict(top_k=V - 1, top_p=0.5, min_p=0.01)):
        check_sample(ctx, rows, u, **how)


def test_scores_under_capture_need_a_first_call(ctx):
    g = gen(41)
    W, X = torch.randn(70, 40, generator=g), torch.randn(500, 40, generator=g).cuda()
    ctx.set_prototypes(W.numpy())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(VqhipError) as e:
        with torch.cuda.graph(graph):
            ctx.scores(X)
    assert e.value.code == _lib.ERR_STATE
    torch.cuda.synchronize()
    want = ctx.scores(X)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ctx.scores(X)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    ctx.set_prototypes((W * 2).numpy())                         # the layout follows the model
    assert (wide(ctx.scores(X)) - ref.scores(X.cpu().numpy(), 2 * W.numpy())).max() < 1e-3


def test_contexts_and_streams_at_the_same_time():
    g = gen(42)
    W = [torch.randn(300, 64, generator=g), torch.randn(200, 64, generator=g)]
    X, u = torch.randn(4000, 64, generator=g).cuda(), torch.rand(4000, generator=g).cuda()
    contexts = [Context(0), Context(0)]
    want = []
    for c, w in zip(contexts, W):
        c.set_prototypes(w.numpy())
        idx, prob = c.assign_sampled(X, u, temperature=20.0)
        want.append((idx, prob, c.lookup(idx), c.lookup_gradient(X, idx)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                idx, prob = contexts[k].assign_sampled(X, u, temperature=20.0)
                got[k].append((idx, prob, contexts[k].lookup(idx), contexts[k].lookup_gradient(X, idx)))
    torch.cuda.synchronize()
    for k in (0, 1):
        for one in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[k]))
    for c in contexts:
        c.close()


def test_offsets_beyond_32_bits(ctx):
    """Rows more than 2^31 elements apart: tables, results and scores that lie far from each other in one allocation of 9 GB."""
    g = gen(43)
    far = (1 << 31) + 17
    buf = torch.zeros(2 * far + 64, dtype=torch.float16, device="cuda")
    rows = buf.as_strided((3, 50), (far, 1))
    values = torch.randn(3, 50, generator=g).half()
    rows.copy_(values.cuda())
    check_sample(ctx, values, torch.tensor([0.2, 0.5, 0.9]), dev=rows, top_p=0.8)
    idx = torch.tensor([2, 0, 1, 2], dtype=torch.int32)
    assert torch.equal(ctx.lookup(idx.cuda(), table=rows).cpu(), values[idx.long()])
    check_gradient(ctx, values, torch.tensor([1, 0, 1], dtype=torch.int32), 4, dev=rows)
    rows.zero_()
    out = ctx.lookup(idx[:3].cuda(), table=values.cuda(), out=rows)
    assert torch.equal(out.cpu(), values[idx[:3].long()])
    G = ctx.lookup_gradient(values.cuda(), idx[:3].cuda(), K=3, out=rows)
    want = torch.zeros(3, 50).half().index_add_(0, idx[:3].long(), values)
    assert torch.equal(G.cpu(), want)
    del rows, out, G
    for D in (8, 40):
        W, X = torch.randn(30, D, generator=g), torch.randn(3, D, generator=g)
        ctx.set_prototypes(W.numpy())
        near = ctx.scores(X.cuda())
        out = buf.view(torch.float32)
        far32 = (1 << 30) + 9
        out = out.as_strided((3, 30), (far32, 1))
        ctx.scores(X.cuda(), out=out)
        assert torch.equal(out, near)
    del buf, out
    torch.cuda.empty_cache()


def test_many_rows_and_few(ctx):
    """More rows than workgroups or waves are launched for (the kernels walk on), and single ones."""
    g = gen(44)
    rows = torch.randn(70000, 5, generator=g)
    u = torch.rand(70000, generator=g)
    idx, _ = ctx.sample(rows.cuda(), u.cuda(), top_k=3)
    for i in (0, 1, 65535, 65536, 69999):
        assert idx[i].item() == ref.sample_row(rows[i].numpy(), u[i].item(), top_k=3)[0]
    a, b = ctx.sample(rows.cuda(), u.cuda(), top_p=0.7)
    c, d = ctx.sample(rows[-7:].cuda(), u[-7:].cuda(), top_p=0.7)
    assert torch.equal(a[-7:], c) and torch.equal(b[-7:], d)


@pytest.mark.parametrize("K,D", [(2000, 2), (1 << 20, 1), (600000, 16), (1, 1)])
def test_gradient_of_very_many_rows(ctx, K, D):
    """Above four million rows the sort takes larger tiles; K: 11 digits in one pass, two passes, a table cleared beside the sort, one."""
    g, N = gen(K), (4 << 20) + 70003
    grad = torch.randint(-8, 9, (N, D), generator=g).half()                # sums of whole numbers: every order gives the same
    idx = (torch.rand(N, generator=g) ** 2 * (K + 1)).int() - 1
    G, counts = ctx.lookup_gradient(grad.cuda(), idx.cuda(), K=K, out_dtype=torch.float32, want_counts=True)
    named = idx >= 0
    want = torch.zeros(K, D, dtype=torch.float64).index_add_(0, idx[named].long(), grad[named].double())
    assert want.abs().max() < 2 ** 24
    assert torch.equal(G.cpu().double(), want)
    assert torch.equal(counts.cpu().long(), torch.bincount(idx[named].long(), minlength=K))


def test_widest_rows(ctx):
    D = (1 << 22) - 1                                                       # odd: rows of no common alignment
    T = torch.arange(2 * D, dtype=torch.int32).remainder(251).half().view(2, D).cuda()
    idx = torch.tensor([1, 0, -1, 1], dtype=torch.int32, device="cuda")
    Y = ctx.lookup(idx, table=T)
    assert torch.equal(Y[0], T[1]) and torch.equal(Y[1], T[0]) and not Y[2].any() and torch.equal(Y[3], T[1])
    G = ctx.lookup_gradient(Y, idx, K=3, out_dtype=torch.float16)
    assert torch.equal(G[1], 2 * T[1]) and torch.equal(G[0], T[0]) and not G[2].any()
    L, need = _lib.lib(), C.c_size_t(0)
    for D, code in ((1 << 22, _lib.OK), ((1 << 22) + 1, _lib.ERR_INVALID)):
        assert L.vqhip_lookup_gradient_workspace(ctx._h, 4, 3, D, need) == code
        assert L.vqhip_lookup_device(ctx._h, T.data_ptr(), _lib.F16, 1, D, D, idx.data_ptr(), 0, 1.0, Y.data_ptr(), D, None) == code


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_very_long_rows(ctx, dtype):
    """Long beyond every vocabulary: spread ones, and all of them equal, where the order among equal ones decides."""
    g, V = gen(45), 500_009
    rows = torch.stack([torch.randn(V, generator=g) * 4, torch.full((V,), -2.5)]).to(TYPES[dtype])
    u = torch.tensor([0.37, 0.61])
    for how in (dict(), dict(top_p=0.9), dict(top_k=100000, top_p=0.5), dict(top_k=200), dict(min_p=0.05)):
        check_sample(ctx, rows, u, **how)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [1100, 9001])
def test_sample_cuts_beyond_the_list(ctx, V, dtype):
    """Counts above what a list of the largest holds, alone and before a nucleus, among spread scores, few values, values around
    zero and values that are all in one power of two."""
    g = gen(V + 1)
    least = torch.finfo(TYPES[dtype]).smallest_normal
    tiny = torch.tensor([0.0, -0.0, least, -least, least / 4, -least / 4])
    rows = torch.stack([torch.randn(V, generator=g) * 3, torch.randint(-3, 3, (V,), generator=g).float(), tiny[torch.randint(0, 6, (V,), generator=g)],
                        1.0 + torch.rand(V, generator=g), -1.0 - torch.rand(V, generator=g) * 2.0 ** -6]).to(TYPES[dtype])
    rows[:, 11:: 13] = -INF
    u = torch.tensor([0.05, 0.5, 0.8, 0.97, 0.3])
    for how in (dict(top_k=209), dict(top_k=353), dict(top_k=600), dict(top_k=V - 200), dict(top_k=V - 1), dict(top_k=600, top_p=0.9), dict(top_k=600, top_p=0.999),
                dict(top_k=900, top_p=0.3), dict(top_k=208, top_p=0.7)):
        check_sample(ctx, rows, u, **how)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,V", [(5, 65), (5, 128), (5, 129), (5, 257), (5, 511), (5, 512), (5, 513), (3, 8192), (3, 8193), (3, 32768), (3, 32769), (258, 40000), (3, 65537)])
def test_sample_where_the_kernels_change(ctx, N, V, dtype):
    g = gen(V + N)
    rows = (torch.randn(N, V, generator=g) * 3).to(TYPES[dtype])
    u = torch.rand(N, generator=g)
    for how in (dict(), dict(top_k=50, top_p=0.9), dict(top_k=250), dict(top_k=300), dict(top_p=0.8, min_p=0.001)):
        if N <= 5:
            check_sample(ctx, rows, u, **how)
        else:                                                # a few of many rows
            idx, prob = ctx.sample(rows.cuda(), u.cuda(), **how)
            some = torch.tensor([0, 100, N - 1])
            one = ctx.sample(rows[some].cuda(), u[some].cuda(), **how)
            assert torch.equal(idx[some.cuda()], one[0]) and torch.allclose(prob[some.cuda()], one[1], rtol=2e-7, atol=0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [1, 3, 4, 5, 15, 16, 17, 31, 32, 33, 50, 63, 64])
@pytest.mark.parametrize("pad", [0, 3])
def test_sample_short_rows(ctx, V, dtype, pad):
    """Many short rows in one wave, each with its own parameters, ties, masks, infinities and nothing at all."""
    g, N = gen(V), 131
    rows = torch.randn(N, V, generator=g) * 3
    rows[::4] = torch.randint(-2, 3, (len(rows[::4]), V), generator=g).float()
    rows[1::5] = torch.where(torch.rand(len(rows[1::5]), V, generator=g) < 0.5, -INF, rows[1::5])
    rows[2::11], rows[3::13, V // 2], rows[5::17, 0], rows[7::19] = -INF, INF, NAN, torch.finfo(TYPES[dtype]).min
    rows[8::23] += 1e4
    rows = rows.to(TYPES[dtype])
    u = torch.rand(N, generator=g)
    buf = torch.full((N, V + pad), 7.0, dtype=TYPES[dtype]).cuda()
    dev = buf[:, :V]
    dev.copy_(rows.cuda())
    for how in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(top_k=5, top_p=0.9, min_p=0.05, temperature=0.3), dict(temperature=50.0, top_p=0.99),
                dict(temperature=1e-3, top_p=0.5), dict(top_p=0.9999999)):
        check_sample(ctx, rows, u, dev=dev, **how)
    per = dict(temperature=torch.rand(N, generator=g) * 2 * (torch.rand(N, generator=g) > 0.2), top_k=torch.randint(0, V + 2, (N,), generator=g).int(),
               top_p=torch.rand(N, generator=g) * 1.2, min_p=torch.rand(N, generator=g) * 0.3)
    check_sample(ctx, rows, u, dev=dev, **per)


def test_every_kernel_in_graphs(ctx):
    """Each size class in two captured graphs, replayed in turn with eager work between and inputs that change in place."""
    g = gen(46)
    rows = [torch.randn(9, V, generator=g).cuda() * 3 for V in (10, 30, 64, 100, 200, 400, 1000, 3000, 20000, 70000)]
    u = torch.rand(9, generator=g).cuda()
    X = [torch.randn(N, 16, generator=g).cuda() for N in (5, 300)]
    grads = [(torch.randn(N, D, generator=g).cuda(), torch.randint(-1, K, (N,), generator=g).int().cuda(), K) for N, K, D in
             ((50, 40, 6), (6000, 40, 6), (9000, 3000, 4), (700, 20000, 512), (9000, 20000, 512), (6000, 20000, 512))]
    models = [torch.randn(K, 16, generator=g).numpy() for K in (7, 90)]
    ctx.set_prototypes(models[1])

    def work():
        out = []
        for r in rows:
            out += ctx.sample(r, u, top_k=40, top_p=0.9) + ctx.sample(r, u, top_p=0.8) + ctx.sample(r, u, top_k=600, min_p=0.01)
        for x in X:
            out += [ctx.scores(x), *ctx.assign_sampled(x, u[:1].expand(len(x)).contiguous())]
        for G, idx, K in grads:
            out += [*ctx.lookup_gradient(G, idx, K=K, want_counts=True), ctx.lookup(idx, table=G)]
        return out

    work()
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(work())
    for step in range(3):
        for r in rows:
            r.mul_(0.9).add_(torch.randn(r.shape, generator=g).cuda())
        for G, idx, K in grads:
            G.neg_()
            idx.copy_(torch.randint(-1, K, (len(idx),), generator=g).int())
        want = work()
        torch.cuda.synchronize()
        for graph, out in zip(graphs, held):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), step
            work()


@pytest.mark.parametrize("K,D", [(3, 4), (16, 16), (31, 4), (40, 12), (64, 3), (100, 16), (20, 30), (300, 20)])
def test_scores_do_not_depend_on_the_rows_beside(ctx, K, D):
    """What the chunks of assign_sampled rest on.  Up to 16 values the same bits; beyond, a close pair is measured alone or with a
    whole tile, two orders of the same D terms of one sign: at most 2 (D + 3) 2^-24 of the distance apart."""
    g = gen(K + D)
    W, X = torch.randn(K, D, generator=g), torch.randn(700, D, generator=g)
    X[::7] = W[torch.randint(K, (100,), generator=g)] + 0.05 * torch.randn(100, D, generator=g)
    X = X.cuda()
    ctx.set_prototypes(W.numpy())
    S = ctx.scores(X)
    for a, b in ((0, 1), (1, 2), (100, 613), (699, 700)):
        part = ctx.scores(X[a:b].contiguous())
        if D <= 16:
            assert torch.equal(part, S[a:b])
        else:
            assert ((part - S[a:b]).abs() <= 2 * (D + 3) * 2.0 ** -24 * S[a:b].abs()).all()
