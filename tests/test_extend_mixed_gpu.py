"""kv800.extend with few queries a row over batches of mixed context on a quantized layer: rows without a sub-block (exact tiles
alone) among rows with many, several of them in one CTA's part of the work, against the definition in 64 bits and with a clean
status word.  Exact tiles lie in the memory that quantized tiles' copies go to, so a part that changes from one kind to the other
has to hand that memory over between the four heads, however many rows apart they are."""
import numpy as np
import pytest
import torch

from test_extend_gpu import Case, close, status_of

SMS = 148      # parts the work is cut into


def batch(rows, limit, most, seed):
    rs = np.random.RandomState(seed)
    return rs.randint(0, limit, rows).tolist(), rs.randint(1, most + 1, rows).tolist()


def chains(rows, most, seed):
    """Runs of rows without a sub-block, up to 15 in a row, each run followed by a row that has some."""
    rs = np.random.RandomState(seed)
    n0 = rs.randint(0, 250, rows)
    at = np.cumsum(rs.randint(2, 16, rows))
    n0[at[at < rows]] = rs.randint(384, 1000, int((at < rows).sum()))
    return n0.tolist(), rs.randint(1, most + 1, rows).tolist()


def handovers(n0, ql):
    """How many parts hold two or more segments with exact tiles and a later one that begins with quantized tiles."""
    items, W = [], 0
    for a, q in zip(n0, ql):
        nq = max(0, a - 128) // 256
        quant = 2 * nq
        tiles = quant + -(-(a + q - 256 * nq) // 128)
        items.append((W + 1, quant, tiles))          # a unit for the item's beginning, then its key tiles
        W += 1 + tiles
    q, rem = divmod(W, SMS)
    found = 0
    for c in range(SMS):
        u0, u1 = (x * q + min(x, rem) for x in (c, c + 1))
        exact = 0
        for b, quant, tiles in items:
            t0, t1 = max(u0 - b, 0), min(u1 - b, tiles)
            if t0 >= t1:
                continue
            if t0 < quant and exact >= 2:
                found += 1
                break
            exact = (0 if t0 < quant else exact) + (t1 > quant)
    return found


BATCHES = [batch(64, 4000, 6, 2), batch(64, 4000, 5, 4), batch(256, 1000, 6, 1), batch(256, 4000, 4, 2), batch(512, 1000, 5, 3), batch(512, 4000, 6, 4),
           batch(513, 1000, 6, 5), batch(2048, 1000, 3, 6), chains(500, 4, 7), chains(1500, 6, 8)]
IDS = [f"{len(a)} rows below {max(a) + 1}, {max(q)}" for a, q in BATCHES]


@pytest.mark.parametrize("n0,ql", BATCHES, ids=IDS)
def test_batches_hand_over(n0, ql):
    """The batches have what they are here for (no GPU)."""
    assert handovers(n0, ql) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("n0,ql", BATCHES, ids=IDS)
def test_mixed_context(n0, ql):
    c = Case("quant", n0, ql, ebs=16, seed=len(n0))
    ref = c.ref()
    for _ in range(3):
        out, status = status_of(c.paged(), c.q, c.qsl, c.cos, c.sin, max(ql))
        assert status == 0
        close(out, ref)


@pytest.mark.gpu
def test_mixed_context_repeats():
    """Which head is ahead does not show: the same bits every time."""
    c = Case("quant", *chains(900, 5, 9), ebs=16, seed=9)
    a = c.run()
    for _ in range(20):
        assert torch.equal(a, c.run())
