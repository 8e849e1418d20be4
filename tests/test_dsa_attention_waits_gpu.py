"""dsa_paged_attention when a copy is given up: the row becomes NaN, the status
says so, the copies in flight are drained, and the calls before and after are
untouched. The first warp of every row takes a wait as run out while its copies
complete as ever: no copy is lost and nothing hangs."""
import math

import pytest
import torch

from oracle import kv_oracle as R
from flagos_kernelgen_72h_shanghai_2026_b200 import dsa_paged_attention
from test_dsa_attention_gpu import E4M3, INT8, check, dev, inputs  # noqa: F401
from test_dsa_attention_range_gpu import check as check_range

pytestmark = pytest.mark.gpu

# B, Q, K, G, D, block_size, code: a CTA to a row and clusters of CTAs, four chunks and more to a warp, blocks of one
# chunk, of two and of a half
SHAPES = [(19, 16, 16, 4, 128, 64, E4M3), (19, 16, 16, 16, 128, 64, E4M3), (1, 1, 128, 4, 128, 64, E4M3),
          (1, 1, 128, 16, 64, 64, INT8), (1, 1, 128, 8, 256, 64, E4M3), (1, 2, 250, 16, 256, 16, INT8)]


def call(dev, x, **kw):
    q, c, blocks, pages, pos, lens = x
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:3], 7.0, device=dev)
    dsa_paged_attention(q, *c, blocks, pages, pos, lens, out, lse, 0.1, **kw)
    return out, lse


@pytest.mark.parametrize("B,Q,K,G,D,bs,code", SHAPES, ids=str)
def test_a_wait_that_runs_out(dev, B, Q, K, G, D, bs, code):
    _, table, _, c, q, _, _, pos, lens = inputs(100 + K, B=B, Q=Q, G=G, D=D, bs=bs, K=K, NB=K, code=code)
    blocks = torch.arange(K).expand(B, 2, Q, K).int().contiguous()
    pages = table[:, None, None, :].expand(B, 2, Q, K).contiguous()
    pos[:] = lens[:, None] - 1
    if Q > 1:
        pos[0, 1] = -1  # a row without tokens has no copy to wait for
    x = [t.to(dev) for t in (q, blocks, pages, pos, lens)]
    x = (x[0], [t.to(dev) for t in c], *x[1:])
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    want = call(dev, x, status=status)
    assert int(status) == 0
    if B * Q <= 4:
        check(*want, R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1), D, R.QMAX[code])
    full = torch.ones(B, Q, dtype=torch.bool)
    full[pos < 0] = False
    # keys' and values' waits of the first chunk and of later ones
    for copies in (2, 3, 4, 5, 6, 7):
        status.zero_()
        bad = call(dev, x, status=status, _test_copies=copies)
        good = call(dev, x, status=torch.zeros_like(status))
        assert int(status) == 9, copies
        for t in bad:
            assert t[full].isnan().all(), copies
        assert (bad[0][~full] == 0).all() and (bad[1][~full] == -math.inf).all()
        for t, w in zip(good, want):
            assert torch.equal(t, w), copies
    # one after the other with nothing between, the last one sound
    for _ in range(20):
        call(dev, x, _test_copies=3)
        good = call(dev, x)
    for t, w in zip(good, want):
        assert torch.equal(t, w)


def test_rows_that_do_not_come_so_far(dev):
    """Nobody starts so many copies: nothing runs out. (The row goes through the copy of the kernel's loop in which waits
    are given up, whose sums are those of value scales far apart.)"""
    _, _, _, c, q, blocks, pages, pos, lens = inputs(101)
    x = [t.to(dev) for t in (q, blocks, pages, pos, lens)]
    x = (x[0], [t.to(dev) for t in c], *x[1:])
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = call(dev, x, status=status, _test_copies=1000)
    assert int(status) == 0
    check_range(*got, R.dsa_paged_attention_ref(q, *c, blocks, pages, pos, lens, 0.1), 128, 448.0)


def test_refusals(dev):
    _, _, _, c, q, blocks, pages, pos, lens = inputs(102)
    x = [t.to(dev) for t in (q, blocks, pages, pos, lens)]
    x = (x[0], [t.to(dev) for t in c], *x[1:])
    for bad, err in ((torch.zeros(1, dtype=torch.int64, device=dev), TypeError), (torch.zeros(1, dtype=torch.int32), TypeError),
                     (torch.zeros(2, dtype=torch.int32, device=dev), ValueError)):
        with pytest.raises(err):
            call(dev, x, status=bad)
    for copies in (-1, 1):
        with pytest.raises(ValueError):
            call(dev, x, _test_copies=copies)
