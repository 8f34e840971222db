"""vqhip_sample_device: rows longer than a wave holds, where sums are put together from many parts."""
import math

import numpy as np
import pytest
import torch

import codes_reference as ref
from vq_amd import Context, _lib

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


# ---------------------------------------------------------------------------------------------- long flat tails
def flat_tail(V, tail, top_p, u, levels=1, top_k=0):
    """One score of 0 and behind it V - 1 of weight w (or halves of two weights, the larger first) each too small to count beside the
    first, but not together -> (index, probability, distance of what decides them from the next index), all in 64 bits."""
    tails = [np.float32(tail), np.float32(tail - 0.25)][:levels]
    w = [math.exp(float(t)) for t in tails]
    n = [(V - 1) // levels] * (levels - 1)
    n.append(V - 1 - sum(n))
    if top_k:
        left = top_k - 1
        n = [min(k, max(0, left - sum(n[:i]))) for i, k in enumerate(n)]
    p, u = float(np.float32(top_p)), float(np.float32(u))
    room = p * (1.0 + sum(a * b for a, b in zip(n, w))) - 1.0            # mass of the tail that is kept
    kept, margin = [], math.inf
    for k, x in zip(n, w):
        r = max(0, min(k, math.ceil(room / x)))
        if 0 < r < k:
            margin = min(margin, abs(room / x - round(room / x)))
        kept.append(r)
        room -= k * x
    total = 1.0 + sum(a * b for a, b in zip(kept, w))
    past = u * total - 1.0
    if past < 0:
        return 0, 1.0 / total, margin
    at = 1
    for r, x in zip(kept, w):
        if past < r * x:
            q = past / x
            return at + math.floor(q), x / total, min(margin, abs(q - round(q)))
        past -= r * x
        at += r
    raise AssertionError("u is below 1")


@pytest.mark.parametrize("levels", [1, 2])
@pytest.mark.parametrize("V,tail,top_p", [(1 << 22, -28.75, 1 - 2.0 ** -20), (1 << 22, -28.75, 1 - 2.0 ** -21), (1 << 24, -26.0, 1 - 2.0 ** -16), ((1 << 24) + 77, -24.0, 0.9999)])
def test_a_long_flat_tail_counts(ctx, V, tail, top_p, levels):
    """Tails that weigh 1e-6 of the row and more, of weights below 2^-38 each."""
    row = torch.empty(1, V, device="cuda")
    row[0, 0] = 0.0
    half = 1 + (V - 1) // levels
    row[0, 1:half] = tail
    row[0, half:] = tail - 0.25
    for u in (0.0, 0.5, 1 - 2.0 ** -22, 1 - 2.0 ** -24):
        for top_k in (0, V // 2 + 5):
            at, prob, margin = flat_tail(V, tail, top_p, u, levels, top_k)
            idx, p = ctx.sample(row, torch.tensor([u], device="cuda"), top_p=top_p, top_k=top_k)
            assert margin > 0.01 or abs(idx.item() - at) <= 1
            assert margin <= 0.01 or idx.item() == at, (u, top_k, idx.item(), at, margin)
            assert abs(p.item() - prob) <= (2.0 ** -24 + 1e-9) * prob


# ---------------------------------------------------------------------------------------------- the same bits wherever a row lies
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H", [15, 31, 60, 127, 250, 501, 1003, 5003, 20001, 40001])
def test_a_draw_does_not_depend_on_where_its_row_begins(ctx, H, dtype):
    """Rows of two equal halves and u = 0.5: the target is the border between them, and the last bit of a sum decides on which side the
    draw falls.  Which side is the sums' affair, but it has to be the same one at every distance from a 16-byte boundary."""
    g = gen(H)
    N = 400 if H <= 5003 else 60
    half = (torch.randn(N, H, generator=g) * 3).to(TYPES[dtype])
    rows = torch.cat([half, half], 1).cuda()
    u = torch.full((N,), 0.5, device="cuda")
    hows = (dict(), dict(temperature=0.7), dict(top_p=0.9), dict(min_p=1e-4), dict(top_k=2 * (H // 3)), dict(top_k=2 * (H // 2), top_p=0.999))
    want = [ctx.sample(rows, u, **how) for how in hows]
    align = 16 // rows.element_size()
    for off in range(1, align + 1):
        buf = torch.full((N, (2 * H + 2 * align) // align * align), 9.0, device="cuda").to(TYPES[dtype])
        moved = buf[:, off:off + 2 * H]
        moved.copy_(rows)
        for how, (idx, prob) in zip(hows, want):
            i, p = ctx.sample(moved, u, **how)
            assert torch.equal(i, idx) and torch.equal(p, prob), (off, how, (i != idx).sum().item(), (p != prob).sum().item())


@pytest.mark.parametrize("H,N,chunks", [(1001, 64, (1, 3, 5, 33)), (5003, 64, (1, 7, 63)), (20001, 300, (1, 100, 256, 257))])
def test_assign_sampled_is_scores_and_sample_for_long_rows(ctx, H, N, chunks):
    """Prototypes twice over and u = 0.5, as above: chunks begin at other distances from a 16-byte boundary than the rows of one
    matrix, and have fewer rows."""
    g = gen(H)
    half, X = torch.randn(H, 3, generator=g), torch.randn(N, 3, generator=g).cuda()
    ctx.set_prototypes(torch.cat([half, half]).numpy())
    u = torch.full((N,), 0.5, device="cuda")
    L = _lib.lib()
    for t, p in ((1.0, 1.0), (2.0, 0.9)):
        idx, prob = ctx.sample(ctx.scores(X), u, temperature=t, top_p=p)
        a, b = ctx.assign_sampled(X, u, temperature=t, top_p=p)
        assert torch.equal(a, idx) and torch.equal(b, prob)
        for rows in chunks:
            work, i, q = torch.empty(rows * 2 * H, device="cuda"), torch.empty_like(idx), torch.empty_like(prob)
            how = _lib.Sampling(t, p, 0.0, 0, None, None, None, None)
            rc = L.vqhip_assign_sampled_device(ctx._h, X.data_ptr(), N, how, u.data_ptr(), i.data_ptr(), q.data_ptr(), work.data_ptr(), rows * 8 * H,
                                               torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and torch.equal(i, idx) and torch.equal(q, prob), (t, p, rows, (i != idx).sum().item())


# ---------------------------------------------------------------------------------------------- more rows than waves
@pytest.mark.parametrize("dtype,V,pad", [("f32", 65, 0), ("f32", 100, 4), ("f32", 256, 0), ("bf16", 250, 3), ("f16", 600, 0), ("f32", 601, 2)])
def test_waves_that_take_several_rows(ctx, V, dtype, pad):
    """A wave per row, 65536 waves at most: rows 65536 apart share one, which asks for the next row while it works on this one.  Parameters
    per row; masked, infinite, greedy and empty rows in between."""
    N = 2 * 65536 + 517
    g = torch.Generator(device="cuda").manual_seed(V)
    t = TYPES[dtype]
    rows = (torch.randn(N, V, generator=g, device="cuda") * 3).to(t)
    rows[torch.rand(N, V, generator=g, device="cuda") < 0.1] = -INF
    rows[3::11] = rows[3::11].round()
    rows[5::97] = -INF
    rows[7::89, V // 2] = INF
    rows[9::83, 0] = NAN
    buf = torch.full((N, V + pad), 7.0, device="cuda", dtype=t)
    dev = buf[:, :V]
    dev.copy_(rows)
    u = torch.rand(N, generator=g, device="cuda")
    pick = torch.rand(N, generator=g, device="cuda")
    how = dict(temperature=torch.where(pick < 0.1, torch.zeros_like(u), 0.25 + pick), top_k=(torch.rand(N, generator=g, device="cuda") * 60).int() * (pick < 0.6).int(),
               top_p=torch.where(pick < 0.3, torch.ones_like(u), 0.5 + pick / 2), min_p=torch.where(pick > 0.8, pick / 10, torch.zeros_like(u)))
    idx, prob = ctx.sample(dev, u, **how)
    for a in range(0, N, 40000):
        b = min(N, a + 40000)
        i, p = ctx.sample(dev[a:b], u[a:b], **{k: v[a:b] for k, v in how.items()})
        assert torch.equal(i, idx[a:b]) and torch.equal(p, prob[a:b]), a
    for i in [0, 1, 5, 7, 9, 65533, 65534, 65535, 65536, 65537, 65541, 131071, 131072, 131073, N - 2, N - 1] + torch.randint(0, N, (200,), generator=gen(V)).tolist():
        one = {k: v[i].item() for k, v in how.items()}
        j, p, margin = ref.sample_row(rows[i].float().cpu().numpy(), u[i].item(), **one)
        if margin > 1e-12:
            assert idx[i].item() == j and abs(prob[i].item() - p) <= (2.0 ** -24 + 1e-9) * p, (i, one)


# ---------------------------------------------------------------------------------------------- temperatures at the ends of f32
@pytest.mark.parametrize("V", [40, 700, 1500, 9001])
@pytest.mark.parametrize("t", [1e-44, 1e-40, 1e-37, 1e-30, 1e30, 1e37, 3e38])
def test_temperatures_of_any_size(ctx, V, t):
    """Scores of the temperature's size, subnormal ones among them, and ones that are far smaller and far larger than it."""
    g = gen(V)
    t = float(np.float32(t))
    like = (torch.randn(4, V, generator=g, dtype=torch.float64) * t).clamp(-3e38, 3e38).float()
    rows = torch.cat([like, like / 1000, torch.randn(2, V, generator=g), torch.full((1, V), -3e38), torch.randn(1, V, generator=g) * 1e38])
    rows[1, ::3] = -INF
    u = torch.rand(len(rows), generator=g)
    for how in (dict(), dict(top_p=0.9), dict(top_p=0.3, top_k=V // 2), dict(top_p=0.999, min_p=0.01), dict(top_k=V - 3, top_p=0.99)):
        idx, prob = ctx.sample(rows.cuda(), u.cuda(), temperature=t, **how)
        for i in range(len(rows)):
            j, p, margin = ref.sample_row(rows[i].numpy(), u[i].item(), temperature=t, **how)
            if margin > 1e-12:
                assert idx[i].item() == j and abs(prob[i].item() - p) <= (2.0 ** -24 + 1e-9) * p, (i, how, idx[i].item(), j, margin)


@pytest.mark.parametrize("V", [40, 700, 1500, 9001])
@pytest.mark.parametrize("t", [1e-44, 1.0, 1e37, 1e38, 3e38])
def test_infinite_scores_at_temperatures_of_any_size(ctx, V, t):
    """A row's infinite scores share it, however small the others are beside the temperature; where they are many, a nucleus ends among them."""
    g = gen(V)
    rows = torch.randn(5, V, generator=g)
    rows[0, V // 2] = INF
    rows[1, ::3] = INF
    rows[2, 5:] = INF
    rows[3, [0, V - 1]] = INF
    rows[4, ::2], rows[4, 1::4] = -INF, INF
    u = torch.tensor([0.5, 0.999, 0.3, 0.75, 0.9])
    for how in (dict(), dict(top_p=0.9), dict(top_p=0.3), dict(top_p=0.999, min_p=0.01), dict(top_k=V // 2, top_p=0.5), dict(top_k=3)):
        idx, prob = ctx.sample(rows.cuda(), u.cuda(), temperature=t, **how)
        for i in range(len(rows)):
            j, p, margin = ref.sample_row(rows[i].numpy(), u[i].item(), temperature=t, **how)
            if margin > 1e-12:
                assert idx[i].item() == j and abs(prob[i].item() - p) <= (2.0 ** -24 + 1e-9) * p, (i, how, idx[i].item(), j, margin)
