"""Speculative steps over the 800h cache without a host sync: the tables of a step from the requests' lengths, the new tokens'
K / V into their pages, attention of last token and drafts, verification, and the flush of what became old enough.

A small random model stands in for the target (an embedding, one quantized and one sliding layer, a vocabulary of 1,000).  It
first answers the prompts one token a step; then the same prompts again with drafts, which are that answer with some tokens
spoiled, so that drafts are kept and rejected.  The drafted step is captured once in a CUDA graph and replayed.

    python examples/speculative_steps.py [--rows 8] [--tokens 120] [--drafts 4] [--spoil 0.2]"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm3-kv800_b200"))
from lfm3_kv800 import kv800, spec, vllm_step  # noqa: E402

DEV, V, EB, WIN = "cuda", 1000, 64, 256
QPAGE, QTOK = 262144, 1280                    # bytes and tokens of a page of sub-blocks


def rope(x, pos, cos, sin):
    """The pairs (d, d + 64), d < 32, rotate; the others have no frequency."""
    c, s = (t[pos].float()[:, None] for t in (cos, sin))
    x = x.float()
    a, b = x[..., :32], x[..., 64:96]
    return torch.cat((a * c - b * s, x[..., 32:64], b * c + a * s, x[..., 96:]), -1).to(torch.bfloat16)


class Server:
    """A model of two layers and its caches for `rows` requests of at most max_len tokens."""

    def __init__(self, rows, max_len):
        g = torch.Generator(device=DEV).manual_seed(0)
        self.emb, self.head = torch.randn(V, 256, generator=g, device=DEV), torch.randn(256, V, generator=g, device=DEV)
        self.w = [torch.randn(256, 24 * 128, generator=g, device=DEV) / 16 for _ in range(2)]
        self.o = [torch.randn(2048, 256, generator=g, device=DEV) / 128 for _ in range(2)]
        self.R, self.nqmax = rows, max_len // 256 + 1
        W, WQ = -(-max_len // EB), -(-max_len // QTOK)

        def pages(width, n, tokens, kind):
            return spec.Pages(torch.zeros(rows, width, dtype=torch.int32, device=DEV), torch.arange(n, device=DEV).int(),
                              spec.page_state(rows, n, DEV), tokens, kind)

        self.exact, self.quant = pages(W, rows * W, EB, "tail"), pages(WQ, rows * WQ, QTOK, "flushed")
        self.slide = pages(W, rows * W, EB, "window")
        self.ev = [torch.zeros(rows * W, 4, EB, 256, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        self.qv = torch.zeros(rows * WQ, QPAGE, dtype=torch.uint8, device=DEV).as_strided(
            (rows * WQ, 2, QTOK, 4, 25), (QPAGE, QTOK * 100, 100, 25, 1))
        self.cos, self.sin, _, _ = vllm_step.tables(torch.device(DEV), max_len)
        self.n0 = torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.none = torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step(self, tokens, qlen, mql, drafts, prompt=False):
        """tokens (T,): each row's last token and its drafts, or its prompt.  -> (tokens, how many) emitted; n0 grows."""
        R, T = self.R, tokens.numel()
        s = spec.step_tables(self.n0, qlen, T, self.exact, self.quant, self.status)
        w = spec.step_tables(self.n0, qlen, T, self.slide, None, self.status)
        x = self.emb[tokens.long()]
        for layer, (p, ev) in enumerate(((s, self.ev[0]), (w, self.ev[1]))):
            y = (x @ self.w[layer]).to(torch.bfloat16).view(T, 24, 128)
            q, k, v = rope(y[:, :16], p.positions, self.cos, self.sin), y[:, 16:20].contiguous(), y[:, 20:].contiguous()
            at = dict(epool=ev, ebs=EB, e_hs=EB * 256, e_ts=256, e_v=128, N=p.N)
            if layer == 0:                                    # quantized layer: keys are kept unrotated
                vllm_step.write_slots(ev, k, v, p.slots, self.status)
                t = vllm_step.decode_tables(self.n0, R, self.exact.table, ev.stride(0), self.quant.table, QPAGE, QTOK, self.nqmax)
                P = kv800.Paged(qpool=self.qv, boff=t["boff"], eoff=t["eoff"], NQ=p.NQ, nqmax=self.nqmax, win=0, **at)
                y = kv800.extend(P, q, p.query_start_loc, self.cos, self.sin, mql, self.status)
            else:                                             # sliding layer: keys are kept rotated, the last 256 are seen
                vllm_step.write_slots(ev, rope(k, p.positions, self.cos, self.sin), v, p.slots, self.status)
                t = vllm_step.decode_tables(self.n0, R, self.slide.table, ev.stride(0))
                P = kv800.Paged(qpool=None, boff=None, eoff=t["eoff"], NQ=self.none, nqmax=0, win=WIN, **at)
                y = kv800.extend(P, q, p.query_start_loc, None, None, mql, self.status)
            x = x + y.float().view(T, 2048) @ self.o[layer]
            x = x / x.square().mean(1, keepdim=True).sqrt()
        spec.commit(s)
        spec.commit(w)
        qsl = s.query_start_loc
        if prompt:                                            # the last row of a prompt gives the first token
            last = qsl[1:].long() - 1
            x, tokens, qsl, drafts = x[last], tokens[last], torch.arange(R + 1, device=DEV).int(), 0
        u = torch.rand(x.shape[0], device=DEV)
        noise = torch.empty(R, V, device=DEV).exponential_()
        out, emitted = spec.verify(x @ self.head, tokens, qsl, u, noise, drafts, temperature=self.none.float(),
                                   status=self.status)
        grown = qlen if prompt else emitted                   # rejected drafts are simply not counted
        n1 = self.n0 + grown
        vllm_step.flush_step(self.ev[0], self.exact.table, self.qv, self.quant.table, n1,
                             torch.nn.functional.pad(grown.cumsum(0).int(), (1, 0)), R * (mql // 256 + 2), self.status)
        self.n0.copy_(n1)
        return out, emitted


def answer(rows, tokens, drafts, script=None):
    """-> (rows, tokens) tokens after random prompts, steps taken, us a step.  script: what the drafts are taken from."""
    max_len = 1024 + tokens * (drafts + 1)                                # a row that is done goes on till all are
    sv = Server(rows, max_len)
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(300, 900, (rows,), generator=g)
    prompt = torch.randint(0, V, (int(lens.sum()),), generator=g).int().to(DEV)
    first, _ = sv.step(prompt, lens.int().to(DEV), int(lens.max()), 0, prompt=True)
    text = torch.zeros(rows, tokens + drafts + 1, dtype=torch.int32, device=DEV)
    text[:, 0] = first[:, 0]
    have = torch.ones(rows, 1, dtype=torch.int64, device=DEV)             # tokens of the answer so far
    ar = torch.arange(drafts + 1, device=DEV)
    qlen = torch.full((rows,), drafts + 1, dtype=torch.int32, device=DEV)

    def one():
        inputs = text.gather(1, have - 1)
        if drafts:
            inputs = torch.cat((inputs, script.gather(1, have + ar[:drafts])), 1)
        out, emitted = sv.step(inputs.view(-1), qlen, drafts + 1, drafts)
        at = (have + ar).clamp_max(tokens + drafts)
        text.scatter_(1, at, torch.where(ar < emitted[:, None], out, text.gather(1, at)))
        have.add_(emitted[:, None]).clamp_max_(tokens)

    state = [sv.n0, have, text, sv.exact.state, sv.quant.state, sv.slide.state]
    keep = [t.clone() for t in state]
    side = torch.cuda.Stream()                                            # a first run for the allocations, then the capture
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
        for t, k in zip(state, keep):
            t.copy_(k)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    t0, t1, steps = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True), 0
    t0.record()
    while steps < tokens and (drafts == 0 or steps % 8 or int(have.min()) < tokens):
        graph.replay()
        steps += 1
    t1.record()
    torch.cuda.synchronize()
    if int(sv.status):
        raise RuntimeError(f"status {int(sv.status)}")
    return text[:, :tokens], steps, t0.elapsed_time(t1) * 1e3 / steps


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--rows", type=int, default=8)
    p.add_argument("--tokens", type=int, default=120)
    p.add_argument("--drafts", type=int, default=4)
    p.add_argument("--spoil", type=float, default=0.2)
    a = p.parse_args()
    plain, n, us = answer(a.rows, a.tokens, 0)
    print(f"one token a step: {n} steps of {us:.0f} us")
    g = torch.Generator(device=DEV).manual_seed(3)
    script = torch.nn.functional.pad(plain, (0, a.drafts + 1))
    bad = torch.rand(script.shape, generator=g, device=DEV) < a.spoil
    script = torch.where(bad, torch.randint(0, V, script.shape, generator=g, device=DEV).int(), script)
    text, m, us = answer(a.rows, a.tokens, a.drafts, script)
    same = (text == plain).int().cumprod(1).sum(1).float().mean()
    print(f"{a.drafts} drafts a step: {m} steps of {us:.0f} us; on average the first {same:.1f} of {a.tokens} tokens agree")
    return plain, text, n, m


if __name__ == "__main__":
    main()
