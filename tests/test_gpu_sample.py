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
