"""vqhip_scores_device and vqhip_assign_sampled_device: the sizes and values where the expanded form of the matrix cores meets the direct
one.  e = 2^-24, a rounding to f32; the bounds of the two forms are those derived in test_gpu_codes.py: (D + 3) e of the distance for the
direct one, 8 (2 D + 6) e of it for the expanded one."""
import time

import numpy as np
import pytest
import torch

from vq_amd import Context, VqhipError, _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def wide(t):
    return t.detach().double().cpu().numpy()


def exact(X, W):
    return -torch.cdist(X.double(), W.double(), compute_mode="donot_use_mm_for_euclid_dist").square().numpy()


# ---------------------------------------------------------------------------------------------- sizes of values
@pytest.mark.parametrize("big", [2.0 ** 60, 1.2e19, 1.5e19, 1.8e19, 2.7e19, 3.6e19])
@pytest.mark.parametrize("K,D", [(2, 40), (5, 40), (5, 100), (70, 33)])
def test_scores_of_values_whose_squares_nearly_overflow(ctx, K, D, big):
    """One prototype with one value near the root of the largest float: the norms around the mean, or only their sum, leave the range of
    f32 where most distances do not.  Where the 64-bit distance is beyond f32 the score is -inf."""
    g = gen(D)
    W, X = torch.randn(K, D, generator=g), torch.randn(9, D, generator=g)
    W[1, 7] = big
    X[3], X[4] = W[0], W[1]
    X[5, 7] = big
    X[6, 7], X[7, 9] = -big, big
    ctx.set_prototypes(W.numpy())
    S, want = wide(ctx.scores(X.cuda())), exact(X, W)
    far = -want > 3.5e38
    near = -want < 3.3e38
    assert (S[far] == -np.inf).all()
    assert np.isfinite(S[near]).all() and (np.abs(S - want)[near] <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)[near]).all()
    assert S[3, 0] == 0.0 and S[4, 1] == 0.0


@pytest.mark.parametrize("power", [-40, -50, -55, -58, -60, -62, -64, -66, -70])
def test_scores_of_values_whose_squares_nearly_vanish(ctx, power):
    """A value's square is below the least normal float from 2^-63 on: every product may lose half a subnormal step, 2^-150, on top of its
    rounding; 4 products a value."""
    g, D = gen(1), 40
    W, X = torch.randn(70, D, generator=g), torch.randn(90, D, generator=g)
    X[::7] = W[3]
    W, X = torch.ldexp(W, torch.tensor(power)), torch.ldexp(X, torch.tensor(power))
    ctx.set_prototypes(W.numpy())
    S, want = wide(ctx.scores(X.cuda())), exact(X, W)
    assert (np.abs(S - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want) + 4 * D * 2.0 ** -150).all()
    assert (S[::7, 3] == 0).all()


# ---------------------------------------------------------------------------------------------- bits that depend on the pair alone
def groups(N, K, D, crowd, seed):
    """Samples and prototypes in `crowd` tight groups, sorted, so that whole tiles hold one group; every 29th sample stands alone."""
    g = gen(seed)
    centre = torch.randn(crowd, D, generator=g)
    W = centre[torch.arange(K) * crowd // K] + 1e-3 * torch.randn(K, D, generator=g)
    X = centre[torch.arange(N) * crowd // N] + 1e-3 * torch.randn(N, D, generator=g)
    X[::29] = torch.randn(len(X[::29]), D, generator=g)
    return X, W


@pytest.mark.parametrize("D", [17, 20, 32, 48, 128, 200])
@pytest.mark.parametrize("K,crowd", [(256, 2), (900, 3), (900, 40)])
def test_a_score_depends_on_its_pair_alone(ctx, K, D, crowd):
    """Tiles where all pairs are close, a part of them and none; other numbers of rows take other tiles, and begin them elsewhere."""
    X, W = groups(9000, K, D, crowd, K + D)
    X = X.cuda()
    ctx.set_prototypes(W.numpy())
    S = ctx.scores(X)
    for a, b in ((0, 1), (8999, 9000), (29, 30), (40, 77), (100, 613), (4000, 8500), (0, 8999)):
        assert torch.equal(ctx.scores(X[a:b].contiguous()), S[a:b]), (a, b)
    want = exact(X.cpu(), W)
    assert (np.abs(wide(S) - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("D", [20, 48])
def test_assign_sampled_is_scores_and_sample_in_every_workspace(ctx, D):
    """Chunks that are no multiple of a tile, shorter and longer than one, and a short last one."""
    N, K = 5000, 900
    X, W = groups(N, K, D, 3, D)
    X, u = X.cuda(), torch.rand(N, generator=gen(D)).cuda()
    ctx.set_prototypes(W.numpy())
    L = _lib.lib()
    for how in (dict(temperature=1e-6), dict(temperature=1.0, top_p=0.9)):
        idx, prob = ctx.sample(ctx.scores(X), u, **how)
        a, b = ctx.assign_sampled(X, u, **how)
        assert torch.equal(a, idx) and torch.equal(b, prob)
        for rows in (7, 100, 513, 1000, 4999):
            work, i, p = torch.empty(rows * K, device="cuda"), torch.empty_like(idx), torch.empty_like(prob)
            call = _lib.Sampling(how["temperature"], how.get("top_p", 1.0), 0.0, 0, None, None, None, None)
            rc = L.vqhip_assign_sampled_device(ctx._h, X.data_ptr(), N, call, u.data_ptr(), i.data_ptr(), p.data_ptr(), work.data_ptr(), rows * K * 4,
                                               torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and torch.equal(i, idx) and torch.equal(p, prob), (how, rows)


# ---------------------------------------------------------------------------------------------- the widest tile
@pytest.mark.parametrize("N,K,D", [(262144 + 3, 256, 20), (140000, 509, 17), (262144 - 128 + 1, 250, 36)])
@pytest.mark.parametrize("kind", ["spread", "few", "groups"])
def test_scores_of_so_many_samples_that_tiles_are_widest(ctx, N, K, D, kind):
    """2048 tiles of 128 x 256 or more.  Spread samples, ones with a close prototype each, and groups that fill whole tiles; the rows at
    both ends, the columns at both ends and every 61st row against 64 bits."""
    if kind == "groups":
        X, W = groups(N, K, D, 2, N)
    else:
        g = gen(N)
        W = torch.rand(K, D, generator=g) * 2 - 1
        X = torch.rand(N, D, generator=g) * 2 - 1
        if kind == "few":
            X = W[torch.randint(K, (N,), generator=g)] + 0.02 * X
    ctx.set_prototypes(W.numpy())
    buf = torch.full((N, K + 3), 7.0, device="cuda")
    S = ctx.scores(X.cuda(), out=buf[:, 1:K + 1])
    assert (buf[:, 0] == 7).all() and (buf[:, K + 1:] == 7).all()
    pick = torch.cat([torch.arange(0, N, 61), torch.arange(200), torch.arange(N - 200, N)])
    want = exact(X[pick], W)
    assert (np.abs(wide(S[pick.cuda()]) - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)).all()
    for cols in ([0, 1, 63, 64, 65, 127, 128, 129, 191, 192, K - 2, K - 1],):
        want = exact(X, W[cols])
        assert (np.abs(wide(S[:, cols]) - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)).all()
    small = ctx.scores(X[1000:1700].cuda())
    assert torch.equal(small, S[1000:1700])


# ---------------------------------------------------------------------------------------------- all six products
@pytest.mark.parametrize("D", [17, 33, 100, 784, 1000])
def test_every_piece_of_every_value_counts(ctx, D):
    """Samples and prototypes with one value each, +-a, of three full bf16 pieces: a product of two such values is a single term, so its
    rounding errors do not grow with D.  The prototypes come in pairs +a, -a: their mean is exactly 0.  With e = 2^-24 and B = x^2 + w^2
    (twice |x w| where both are in the same place and of about one size): the norms e B, the sum of six exact products at most 5 e |x w|, doubled,
    what they leave out (below 2^-26 |x w|, doubled) e |x w|, B itself e B, the last addition e |s| <= 2 e B: 4 e B + 11 e |x w| <= 10 e B.
    A product left out or taken twice, or a piece from another place, is off by 2^-17 |x w| and more, six times as much."""
    g = gen(D)
    a = 1.0 + 0.2 * torch.rand(8192, generator=g)
    p1 = a.bfloat16().float()
    p2 = (a - p1).bfloat16().float()
    p3 = a - p1 - p2
    a = a[(p2.abs() > 0.6 * 2.0 ** -8) & (p3.abs() > 0.6 * 2.0 ** -17)]
    assert len(a) > 50
    W, X = torch.zeros(2 * D, D), torch.zeros(D, D)
    at = torch.arange(D)
    W[2 * at, at] = a[at % len(a)]
    W[2 * at + 1, at] = -a[at % len(a)]
    X[at, at] = a[(at * 7 + 3) % len(a)]
    ctx.set_prototypes(W.numpy())
    S = wide(ctx.scores(X.cuda()))
    want = exact(X, W)
    B = wide(X.double().square().sum(1))[:, None] + wide(W.double().square().sum(1))[None]
    close = np.abs(want) < B / 15                                          # measured directly
    assert (np.abs(S - want)[~close] <= 10 * 2.0 ** -24 * B[~close]).all()
    assert (np.abs(S - want)[close] <= (D + 3) * 2.0 ** -24 * np.abs(want)[close]).all()
    assert close[at, 2 * at].all() and not close[at, 2 * at + 1].any()


@pytest.mark.parametrize("N,D,K", [(300, 128, 256), (70, 784, 100), (130, 1000, 70)])
@pytest.mark.parametrize("offset", [0.0, 100.0])
def test_scores_are_within_the_library_s_bar(ctx, N, D, K, offset):
    """1e-5 of the distance, whatever the length."""
    g = gen(D)
    W = torch.rand(K, D, generator=g) * 2 - 1 + offset
    X = W[torch.randint(K, (N,), generator=g)] + 0.5 * (torch.rand(N, D, generator=g) * 2 - 1)
    ctx.set_prototypes(W.numpy())
    want = exact(X, W)
    assert (np.abs(wide(ctx.scores(X.cuda())) - want) <= 1e-5 * np.abs(want)).all()


# ---------------------------------------------------------------------------------------------- models
def test_scores_follow_the_model(ctx):
    """A model after another, of other sizes, larger and smaller, with few prototypes and many."""
    g = gen(5)
    for K, D in ((70, 40), (70, 40), (300, 100), (3, 4), (9, 33), (2000, 17), (2000, 16), (64, 64)):
        W, X = torch.randn(K, D, generator=g) * 3 + 1, torch.randn(100, D, generator=g)
        ctx.set_prototypes(W.numpy())
        want = exact(X, W)
        assert (np.abs(wide(ctx.scores(X.cuda())) - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)).all()


def test_a_model_costs_a_copy_until_scores_are_asked_for(ctx):
    """Setting prototypes keeps them on the host and brings them to the GPU; what only scores need (their mean, their layout) is made by the
    first scores call.  Four times a copy on each side, at the best of several, leaves room for everything but a pass of arithmetic over them."""
    W = np.random.default_rng(0).random((131072, 64), np.float32)

    def best(f):
        t = []
        for _ in range(7):
            torch.cuda.synchronize()
            at = time.perf_counter()
            f()
            torch.cuda.synchronize()
            t.append(time.perf_counter() - at)
        return min(t)

    assert best(lambda: ctx.set_prototypes(W)) <= 4 * best(lambda: torch.from_numpy(W.copy()).cuda())


# ---------------------------------------------------------------------------------------------- no room for the layout
def test_a_layout_that_finds_no_memory_leaves_nothing_behind():
    """The first scores call of a model needs 6 bytes a prototype value.  Where the card has none left it says so, and neither the next
    operation nor the call itself, once there is room, sees that error again."""
    g = gen(8)
    W, X = torch.rand(1 << 19, 512, generator=g), torch.rand(5, 512, generator=g).cuda()
    out = torch.empty(5, 1 << 19, device="cuda")
    with Context(0) as c:
        c.set_prototypes(W.numpy())
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        held = []
        try:
            for size in (16 << 30, 1 << 30, 128 << 20):                                      # (the layout is 1.6 GB)
                try:
                    while True:
                        held.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
                except torch.OutOfMemoryError:
                    pass
            with pytest.raises(VqhipError) as e:
                c.scores(X, out=out)
            assert e.value.code == _lib.ERR_NOMEM
            assert out.fill_(3.0).eq(3.0).all().item()
        finally:
            held.clear()
            torch.cuda.empty_cache()
        c.scores(X, out=out)
        want = exact(X.cpu(), W[:50])
        assert (np.abs(wide(out[:, :50]) - want) <= 1e-5 * np.abs(want)).all()


# ---------------------------------------------------------------------------------------------- more than a launch holds
def test_scores_of_more_samples_than_a_grid_has_lanes(ctx):
    """2^32 samples and 300 more, a lane each: 34 GB of samples and scores."""
    N = (1 << 32) + 300
    X = torch.zeros(N, 1, device="cuda")
    at = [0, 1 << 30, (1 << 32) - 1, 1 << 32, (1 << 32) + 255, (1 << 32) + 256, N - 1]
    for n, i in enumerate(at):
        X[i] = n + 1.0
    ctx.set_prototypes(np.array([[-2.0]], np.float32))
    S = ctx.scores(X, out=torch.zeros(N, 1, device="cuda"))
    assert [S[i].item() for i in at] == [-(n + 3.0) ** 2 for n in range(len(at))]
    assert sum((part == -4.0).sum().item() for part in S.split(1 << 28)) == N - len(at)
    del X, S
    torch.cuda.empty_cache()


@pytest.mark.parametrize("K,D,N", [((1 << 28) + 70, 1, 3), ((1 << 26) + 5, 17, 2)])
def test_scores_against_very_many_prototypes(ctx, K, D, N):
    """Direct tiles of 64 prototypes beyond 2^22, and a layout whose prototypes are more than a grid has waves."""
    W = np.zeros((K, D), np.float32)
    at = [0, 1, 63, 64, 1 << 26, (1 << 26) + 4, K - 71, K - 70, K - 2, K - 1]
    for n, k in enumerate(at):
        W[k, n % D] = n + 2.0
    ctx.set_prototypes(W)
    X = torch.zeros(N, D)
    X[1] = 1.0
    S = ctx.scores(X.cuda())
    got = S[:, at].cpu()
    want = exact(X, torch.from_numpy(W[at]))
    assert (np.abs(wide(got) - want) <= 8 * (2 * D + 6) * 2.0 ** -24 * np.abs(want)).all()
    assert (S[0] == 0).sum().item() == K - len(set(at)) and ((S[1] + D).abs() <= 1e-4 * D).sum().item() >= K - len(set(at))
    del S
    ctx.set_prototypes(W[:3])                                               # (the large layout is not kept)
    torch.cuda.empty_cache()
