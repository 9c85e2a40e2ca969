"""The roundings of a key in kv800.extend are the decode's: a quantized key to bf16 after dequantizing, then the rotated pairs in 32
bits and to bf16 once (exact keys: once in all).

The reference takes keys rounded just so and goes on in 64 bits, so that what is left is the weights' rounding to bf16 (2^-9 at
most, rms 2^-9 / sqrt 3 = 1.1e-3; 11 bits over quantized keys) and the output's (the same, times 1.5 for mantissas near 1), however
large the scores are: 2.0e-3 of the norm as independent errors, below 2.5e-3; of a single row 2^-9 (sum p |v| / |o| + 1), below 5e-3
where few keys carry it.  A key rounded once more moves a score of standard deviation s by about 2^-9 s / sqrt 3 (4e-3 to 1.1e-2 for
s = 3 to 10, more in the worst rows), beyond both."""
import math

import pytest
import torch

from test_extend_gpu import DEV, NSINK, SUB, WIN, Case

from lfm3_kv800 import kv800

pytestmark = pytest.mark.gpu


def as_decoded(c):
    """c's output with keys rounded as the decode rounds them, from there on in 64 bits."""
    out = torch.zeros(c.q.shape, dtype=torch.float64, device=DEV)
    for b in range(c.R):
        a, e = int(c.qsl[b]), int(c.qsl[b + 1])
        K, V = c.K[b][:c.N[b]].clone(), c.V[b][:c.N[b]].double()
        m = 256 * c.nq[b]
        if m:
            sb = c.qpool.view(-1)[c.boff[b, :c.nq[b], None] + torch.arange(SUB, device=DEV)]
            k, v = kv800.dequantize_blocks(sb)
            K[:m], V[:m] = k.view(m, 4, 128), v.view(m, 4, 128).double()
        pos = torch.arange(c.N[b], device=DEV)
        cs, sn = c.cos[pos].float()[:, None], c.sin[pos].float()[:, None]
        K = K.float()
        x, y = K[..., :32].clone(), K[..., 64:96].clone()
        K[..., :32], K[..., 64:96] = x * cs - y * sn, y * cs + x * sn
        K = K.to(torch.bfloat16).double()
        qp = (c.N[b] - (e - a) + torch.arange(e - a, device=DEV))[:, None]
        seen = pos[None] <= qp
        if c.layer == "window":
            seen &= (pos[None] > qp - WIN) | (pos[None] < NSINK)
        for h in range(16):
            s = c.q[a:e, h].double() @ K[:, h // 4].T / math.sqrt(128)
            out[a:e, h] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ V[:, h // 4]
    return out


@pytest.mark.parametrize("layer,n0,ql", [("quant", [2500, 700], [5, 4]), ("quant", [2500, 700], [90, 33]), ("quant", [2500], [20]),
                                         ("quant", [0], [300]), ("quant", [100, 40], [3, 5]), ("window", [700, 20], [5, 2]), ("window", [700], [200])])
@pytest.mark.parametrize("scale", [2, 4, 8])      # scores of standard deviation about 1.4 times that
def test_keys_are_rounded_as_in_decode(layer, n0, ql, scale):
    c = Case(layer, n0, ql, seed=scale)
    c.q *= scale
    ref, got = as_decoded(c), c.run().double()
    total = float((got - ref).norm() / ref.norm())
    row = float(((got - ref).norm(dim=-1) / ref.norm(dim=-1)).max())
    assert total <= 2.5e-3 and row <= 5e-3, f"total {total:.2e}, a row {row:.2e}"
