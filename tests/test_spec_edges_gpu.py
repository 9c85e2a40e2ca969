"""Inputs at the edges of what spec.verify and spec.step_tables take."""
import numpy as np
import pytest
import torch

from test_spec_gpu import make, run

from lfm3_kv800 import spec

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("V", [9, 700, 5001])
def test_greedy_infinities(dtype, probs, V):
    """Greedy rows with +inf: the first of them is the argmax, whatever the path; NaN are skipped; -inf alone gives nothing."""
    rs = np.random.RandomState(V)
    x = torch.randn(12, V, generator=torch.Generator().manual_seed(V)).to(dtype)
    at = rs.randint(1, V - 1, 12)
    for i in (0, 2, 3, 6):
        x[i, at[i]] = float("inf")
    x[2, at[2] + 1:] = float("inf")                  # several: the first
    x[3, 0] = float("nan")
    x[4] = -float("inf")
    x[5] = torch.finfo(dtype).min                    # equal and finite: the first
    x[7] = float("nan")
    x[8, at[8]] = torch.finfo(dtype).max
    x[9, at[9]], x[9, at[9] + 1] = torch.finfo(dtype).max, float("inf")
    key = x.double().nan_to_num(nan=-np.inf, posinf=np.inf, neginf=-np.inf)
    best = [int(r.argmax()) if r.max() > -np.inf else -1 for r in key]
    for good in (True, False):                       # one draft a row of two target rows
        tok = torch.zeros(12, dtype=torch.int32)
        for b in range(6):
            tok[2 * b + 1] = best[2 * b] if good else (best[2 * b] + 1) % V
        want = []
        for b in range(6):
            if best[2 * b] < 0:
                want.append([-1, -1])
            elif good:
                want.append([best[2 * b], best[2 * b + 1]])
            else:
                want.append([best[2 * b], -1])
        if good:
            tok = tok.clamp_min(0)
        q = torch.full((6, V), 1.0 / V, device=DEV) if probs else None
        t, e = spec.verify(x.to(DEV), tok.to(DEV), torch.arange(0, 13, 2, device=DEV).int(), torch.rand(12, device=DEV),
                           torch.ones(6, V, device=DEV), 1, q, torch.zeros(6, device=DEV))
        assert t.tolist() == want
        assert e.tolist() == [sum(v >= 0 for v in w) for w in want]


def test_no_rows_and_no_tokens():
    """A step of nothing leaves the groups as they are."""
    g = spec.Pages(torch.zeros(0, 4, dtype=torch.int32, device=DEV), torch.arange(8, device=DEV).int(), spec.page_state(0, 8, DEV), 64)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    for quant in (None, spec.Pages(g.table, g.ring, spec.page_state(0, 5, DEV), 1280, "flushed")):
        junk = [torch.full((64,), -1, dtype=d, device=DEV) for d in (torch.int32, torch.int64) for _ in range(8)]
        del junk                                     # what a new buffer is made of
        s = spec.step_tables(none, none, 0, g, quant)
        assert s.query_start_loc.tolist() == [0] and s.exact_state.tolist() == [0, 8]
        spec.commit(s)
        assert g.state.tolist() == [0, 8] and (quant is None or quant.state.tolist() == [0, 5])


@pytest.mark.parametrize("probs", [False, True])
def test_verify_results_hold_no_scratch(probs):
    """A result that is kept does not keep the call's workspace."""
    R, K, V = 8, 4, 60000
    x = torch.randn(R * (K + 1), V, device=DEV)
    q = torch.softmax(torch.randn(R * K, V, device=DEV), -1) if probs else None
    t, e = spec.verify(x, torch.zeros(R * (K + 1), dtype=torch.int32, device=DEV), torch.arange(0, R * (K + 1) + 1, K + 1, device=DEV).int(),
                       torch.rand(R * (K + 1), device=DEV), torch.ones(R, V, device=DEV), K, q)
    for y in (t, e):
        assert y.untyped_storage().nbytes() <= 4 * R * (K + 2) + 512


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("first", [1, 3, 40])
def test_tokens_before_the_first_row(probs, first):
    """query_start_loc that begins above 0: the drafts' probabilities still begin with the first draft's."""
    R, K, V = 9, 3, 801
    x, tok, qsl, u, noise, q, temp = make(R, K, V, torch.float32, probs, 0.2, 11, idle=True)
    want = run(x, tok, qsl, u, noise, K, q, temp)
    pad = lambda t: torch.cat((t[:1].expand(first, *t.shape[1:]), t))  # noqa: E731
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = run(pad(x), pad(tok), qsl + first, pad(u), noise, K, q, temp, st)
    assert int(st) == 0
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
