"""The device work around a chunked or speculative step over the 800h cache, without a host sync: the tables of a step from
the requests' lengths (step_tables) and the verification of drafted tokens (verify).  With kv800.extend between them a step
runs from lengths to new lengths on the device, so it can be captured in a CUDA graph:

    s = spec.step_tables(n0, qlen, T, exact, quant)            # positions, slots, block tables
    vllm_step.write_slots(cache, k, v, s.slots)                # per layer
    out = kv800.extend(paged, q, s.query_start_loc, ...)       # per layer
    tokens, emitted = spec.verify(logits, inputs, s.query_start_loc, u, noise, K, ...)
    spec.commit(s); n0 += emitted                              # rejected drafts are simply not counted

No counterpart in the reference, whose vLLM glue takes these from the engine on the host."""
from dataclasses import dataclass

import torch

from . import _lib
from .kv800 import _check_status, _cuda, _on, _raw_stream, _status_ptr

KINDS = {"all": 0, "tail": 1, "window": 2, "flushed": 3}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_DRAFTS = 63

__all__ = ["Pages", "StepTables", "page_state", "step_tables", "commit", "verify", "KINDS", "MAX_DRAFTS"]


@dataclass
class Pages:
    """A group of pages that the rows of a batch own.

    table  (R, W) int32 page ids, filled in place as rows grow
    ring   (C,) int32: the free ids lie at (head .. tail - 1) % C
    state  int64 [2 R + 2]: pages owned per row | first live column per row | head | tail (page_state() for a new one)
    page_tokens  tokens a page holds
    kind   'all'      every token of a row needs a page, none is given back
           'tail'     exact pages of a quantized layer: those below the flushed sub-blocks go back to the ring
           'window'   exact pages of a window layer: those before the last 255 tokens go back
           'flushed'  pages of sub-blocks: a row needs them for its 256 nq(n) flushed tokens"""
    table: torch.Tensor
    ring: torch.Tensor
    state: torch.Tensor
    page_tokens: int
    kind: str = "all"


@dataclass
class StepTables:
    query_start_loc: torch.Tensor      # (R + 1,) int32
    rows: torch.Tensor                 # (T,) int32, -1 for tokens no row owns
    positions: torch.Tensor            # (T,) int64
    slots: torch.Tensor                # (T,) int64, -1 without a page
    N: torch.Tensor                    # (R,) int32, tokens after the step
    NQ: torch.Tensor                   # (R,) int32, sub-blocks flushed before it
    exact: Pages
    exact_state: torch.Tensor          # int64 [2 R + 2], the group's state once the step is committed
    quant: Pages = None
    quant_state: torch.Tensor = None


def page_state(rows, pages, device):
    """State of `rows` rows without pages over a ring that holds `pages` free ids."""
    s = torch.zeros(2 * rows + 2, dtype=torch.int64, device=device)
    s[-1] = pages
    return s


def _need(t, name, who, dev, dtype, shape=None):
    if t.device != dev:
        _on(t, dev, f"{who} ({name})")
    if t.dtype != dtype or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise ValueError(f"{who}: {name} must be contiguous {dtype}{'' if shape is None else ' ' + str(shape)}, got "
                         f"{t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _group(g, R, dev, out, who):
    table, kind = g.table, KINDS.get(g.kind)
    if kind is None:
        raise ValueError(f"{who}: kind {g.kind!r}: expected one of {', '.join(KINDS)}")
    if table.device != dev:
        _on(table, dev, f"{who} (table)")
    shape = table.shape
    if len(shape) != 2 or shape[0] != R or table.dtype is not torch.int32 or (
            R and (table.stride(1) != 1 or (table.stride(0) < shape[1] and R > 1))):
        raise ValueError(f"{who}: table must be ({R}, W) int32 with rows of its own and unit column stride, got {table.dtype} "
                         f"{tuple(shape)} with strides {table.stride()}")
    return _lib.Pages(table.data_ptr(), max(table.stride(0), shape[1]), shape[1], _need(g.ring, "ring", who, dev, torch.int32),
                      g.ring.numel(), _need(g.state, "state", who, dev, torch.int64, (2 * R + 2,)), out, g.page_tokens, kind)


def step_tables(n0, qlen, max_tokens, exact, quant=None, status=None):
    """Tables of a step in one launch: row r holds n0[r] tokens and takes qlen[r] more (int32, on the device; 0 = idle).
    max_tokens: host bound of their sum, the length of the per-token tables.  New pages come off the rings of `exact` and
    `quant` (a Pages each) in row order, and their tables are filled in place; pages a row no longer needs go back.  The
    groups' states change only with commit(), so a step may be planned again.  status: optional device int32 that
    collects ST_TABLE (8) where a row found no room or the tokens are more than max_tokens.  -> StepTables."""
    dev, R, T = _cuda(n0, "step_tables (n0)").device, n0.numel(), int(max_tokens)
    pn = _need(n0, "n0", "step_tables", dev, torch.int32)
    pl = _need(qlen, "qlen", "step_tables", dev, torch.int32, n0.shape)
    if T < 0:
        raise ValueError(f"step_tables: max_tokens must not be negative, got {max_tokens}")
    pst = _status_ptr(status, dev, "step_tables")
    # the results share two buffers: T positions, T slots, the states | T rows, R + 1 starts, R lengths, R sub-block counts
    n = 2 * R + 2
    m = n if quant is None else 2 * n
    narrow = n0.new_empty(T + 3 * R + 1)
    wide = exact.state.new_empty(2 * T + m)      # int64, or _group refuses
    w, i = wide.data_ptr(), narrow.data_ptr()
    es = w + 16 * T
    ge = _group(exact, R, dev, es, "step_tables: exact")
    gq = None if quant is None else _group(quant, R, dev, es + 8 * n, "step_tables: quant")
    if not R and not T:      # no work for the library: an empty plan, the groups as they are
        narrow.zero_()
        wide[:n].copy_(exact.state)
        if quant is not None:
            wide[n:].copy_(quant.state)
    _lib.call("kv800_step_tables", pn, pl, R, T, ge, gq, i + 4 * T, i, w, w + 8 * T, i + 4 * (T + R + 1),
              i + 4 * (T + 2 * R + 1), pst, _raw_stream(dev.index))
    _check_status(status, dev, "step_tables")
    rows, qsl, N, NQ = narrow.unsafe_split_with_sizes((T, R + 1, R, R))
    pos, slots, est, qst = wide.unsafe_split_with_sizes((T, T, n, m - n))
    return StepTables(qsl, rows, pos, slots, N, NQ, exact, est, quant, None if quant is None else qst)


def commit(s):
    """Make a step's page states the groups' own (device copies on the current stream)."""
    s.exact.state.copy_(s.exact_state)
    if s.quant is not None:
        s.quant.state.copy_(s.quant_state)


def verify(logits, tokens, query_start_loc, uniform, noise, max_drafts, draft_probs=None, temperature=None, status=None):
    """Verification of drafted tokens from given random numbers, two launches.

    logits: (T, V) bf16 / fp16 / fp32 target logits, row b's at query_start_loc[b] .. query_start_loc[b + 1]: one for each
    of its drafts and one after them.  tokens: (T,) int32, the step's input tokens (a row's drafts are all but its first).
    uniform: (T,) fp32 in [0, 1); noise: (R, V) fp32 > 0, exponentially distributed.  draft_probs: (drafts, V) fp32 in
    order, None for certain drafts (a lookup).  temperature: (R,) fp32, 0 = greedy, None = 1.
    -> tokens (R, max_drafts + 1) int32 (the accepted drafts, the next token, -1) and emitted (R,) int32, how many.
    A draft stands while all before it do and u q(d) < p(d); the next token is argmax (p - q)+ / noise where one fell,
    argmax p / noise where all stood: the target's distribution, whatever the drafts were."""
    if not logits.is_cuda:
        _cuda(logits, "verify")
    shape, dtype = logits.shape, _DTYPES.get(logits.dtype)
    if len(shape) != 2 or dtype is None or (shape[0] and logits.stride(1) != 1):
        raise ValueError(f"verify: logits must be (T, V) bf16 / fp16 / fp32 with unit column stride, got {logits.dtype} "
                         f"{tuple(shape)}")
    dev, (T, V) = logits.device, shape
    K, R = int(max_drafts), query_start_loc.numel() - 1
    if R < 0 or K < 0 or V < 1:
        raise ValueError(f"verify: {R} rows, {K} drafts, {V} tokens")
    pt = _need(tokens, "tokens", "verify", dev, torch.int32, (T,))
    ps = _need(query_start_loc, "query_start_loc", "verify", dev, torch.int32, (R + 1,))
    pu = _need(uniform, "uniform", "verify", dev, torch.float32, (T,))
    pt0 = None if temperature is None else _need(temperature, "temperature", "verify", dev, torch.float32, (R,))
    pst = _status_ptr(status, dev, "verify")
    noise, ln = _wide(noise, "noise", dev, R, V)
    nq = lq = pq = None
    if draft_probs is not None:
        nq = draft_probs.shape[0]
        draft_probs, lq = _wide(draft_probs, "draft_probs", dev, nq, V)
        pq = draft_probs.data_ptr() or noise.data_ptr()      # no row at all: any address, none is read
    if T > 1 and logits.stride(0) < V:
        logits = logits.contiguous()                         # rows that overlap (expanded)
    words = _lib.lib().kv800_verify_workspace_size(R, min(K, MAX_DRAFTS), V) >> 2
    scratch, buf = tokens.new_empty(words), tokens.new_empty(R * (K + 2))      # buf: tokens, counts
    p, n = buf.data_ptr(), R * (K + 1)
    _lib.call("kv800_verify", logits.data_ptr(), dtype, max(logits.stride(0), V), T, V, pt, ps, R, K, pu, noise.data_ptr(), ln,
              pq, nq or 0, lq or 0, pt0, p, p + 4 * n, scratch.data_ptr(), 4 * words, pst, _raw_stream(dev.index))
    out, emitted = buf.unsafe_split_with_sizes((n, R))
    out = out.view(R, K + 1)
    _check_status(status, dev, "verify")
    return out, emitted


def _wide(t, name, dev, rows, V):
    """A (rows, V) fp32 tensor whose rows do not overlap, and their stride."""
    if t.device != dev:
        _on(t, dev, f"verify ({name})")
    if t.dtype != torch.float32 or t.shape != (rows, V) or (rows and t.stride(1) != 1):
        raise ValueError(f"verify: {name} must be ({rows}, {V}) fp32 with unit column stride, got {t.dtype} {tuple(t.shape)}")
    if rows > 1 and t.stride(0) < V:
        t = t.contiguous()
    return t, max(t.stride(0), V)
