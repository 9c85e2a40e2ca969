"""Inputs at the edges of what kv800.extend takes."""
import ctypes

import pytest
import torch

import test_extend_gpu as base
from test_extend_gpu import DEV, Case, close

from lfm3_kv800 import _lib, kv800

pytestmark = pytest.mark.gpu


def filled(c, maxq=None, value=float("nan")):
    """(output, status word) of a call through the C entry into a buffer that holds `value`."""
    P = c.paged()
    s, keep = kv800._paged_struct(P, c.q.device, c.qsl.numel() - 1)
    out = torch.full_like(c.q, value)
    R, T, maxq = c.qsl.numel() - 1, c.q.shape[0], maxq or max(1, max(c.ql))
    n = _lib.lib().kv800_extend_workspace_size(R, T, maxq)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV)
    cs, sn = (None, None) if c.layer == "slide" else (c.cos.data_ptr(), c.sin.data_ptr())
    _lib.call("kv800_extend", ctypes.byref(s), c.q.data_ptr(), c.qsl.data_ptr(), R, T, maxq, cs, sn, c.cos.shape[0], out.data_ptr(),
              ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out, int(ws[:4].view(torch.int32))


@pytest.mark.parametrize("at", [49152, 49664])      # V offsets, V scales
@pytest.mark.parametrize("n0,ql", [(252, 5), (250, 8), (230, 30), (200, 90)])
def test_nan_scale_of_a_hidden_key(n0, ql, at):
    """A V scale or offset that is NaN makes those queries NaN that see its key, in a sub-block that reaches past others."""
    c = Case("quant", [n0], [ql], nq=[1], seed=ql)
    ref = c.ref()
    first = n0 + ql // 2                            # tokens from here on
    c.qpool[0, at + 2 * first:at + 512] = 0x7f
    out, status = filled(c)
    assert status == 0
    close(out[:ql // 2], ref[:ql // 2])
    assert torch.isnan(out[ql // 2:]).all()


@pytest.mark.parametrize("layer", ["quant", "window", "slide"])
@pytest.mark.parametrize("ql", [[4, 0, 2], [60, 3, 20]])
def test_tokens_before_the_first_row(layer, ql):
    """query_start_loc that begins above 0: no row owns the tokens before it, they get zeros."""
    c = Case(layer, [500, 30, 9], ql, pad=10, seed=2)
    ref = c.ref()
    c.qsl += 7
    c.q = torch.roll(c.q, 7, 0)
    out, status = filled(c)
    n = sum(ql)
    assert status == 0 and (out[:7] == 0).all() and (out[n + 7:] == 0).all()
    close(out[7:n + 7], ref[:n])


@pytest.mark.parametrize("n0,ql", [([900], [5]), ([900], [90]), ([520, 40], [40, 200]), ([600, 90], [1, 3])])
@pytest.mark.parametrize("sinks", [100, 128, 129, 200, 300])
def test_many_sinks(monkeypatch, n0, ql, sinks):
    """Any number of sinks, those past a tile among them, each rotated by its own position."""
    monkeypatch.setattr(base, "NSINK", sinks)
    monkeypatch.setattr(kv800, "NSINK", sinks)
    c = Case("window", n0, ql, seed=sinks)
    out, status = filled(c)
    assert status == 0
    close(out, c.ref())


@pytest.mark.parametrize("layer", ["window", "slide"])
@pytest.mark.parametrize("win", [300, 2 ** 31 - 100, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 62])
@pytest.mark.parametrize("ql", [5, 90])
def test_wide_windows(monkeypatch, layer, win, ql):
    """A window beyond the row's length, or beyond 32 bits, hides nothing."""
    monkeypatch.setattr(base, "WIN", win)
    c = Case(layer, [700, 3], [ql, 2], seed=ql)
    out, status = filled(c)
    assert status == 0
    close(out, c.ref())


@pytest.mark.parametrize("ql", [5, 90])
def test_status_reaches_the_caller(ql):
    """A range check that fires inside the call shows in the caller's status word, beside the bits it held, in a graph too."""
    c = Case("quant", [1500], [ql], seed=16)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    call = lambda P, status=st: kv800.extend(P, c.q, c.qsl, c.cos, c.sin, ql, status)  # noqa: E731
    assert torch.equal(call(c.paged()), c.run()) and int(st) == 0
    P = c.paged()
    P.boff = c.boff.clone()
    P.boff[0, 1] = c.qpool.numel()
    call(P)
    assert int(st) == 1
    P = c.paged()
    P.eoff = c.eoff.clone()
    P.eoff[0, -1] = c.epool.numel() - 8
    call(P)
    assert int(st) == 3
    call(c.paged())
    assert int(st) == 3
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(P)
    st.zero_()
    g.replay()
    assert int(st) == 2
