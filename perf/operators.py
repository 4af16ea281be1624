"""Operators of a serving step with several new tokens per sequence, as a user calls them, with what each has to move and compute
and what its results are in 64 bits.

Kinds of cases (a case is a dict of plain values, see `listed`):

  append   `ops.paged_kv_append_rope`: the new tokens of a packed batch of sequences are rotated to their positions (one position per
           token, or one per axis: time, height and width of images and video) and their keys and values written to the pages
           behind what each sequence holds; the rotated queries come back.
  chunk    `ops.paged_gqa_attention_chunk`: causal attention of each sequence's new tokens over everything its pages hold, new tokens
           included, with or without a sigmoid gate on the output.  One token per sequence is the decode step, a few are
           the check of a speculated continuation, hundreds are a portion of a prompt.
  sample   `ops.sample_rows`: the next token of every row of logits, by temperature, top-k, min-p and top-p of the row's own, from
           given random numbers.

Lengths belong to the case, values to the seed.  8 query heads on 2 key/value heads of 256 with 64 rotated dimensions, pages of 16
tokens, vocabularies of 248320 and 65536 are this repository's own; the other head layouts and vocabularies are generic.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV, BF, F32, F64 = "cuda", torch.bfloat16, torch.float32, torch.float64
PAGE, THETA = 16, 1e7


def _ops():
    root = str(Path(__file__).resolve().parent.parent / "qwen3_5-triton-inference-engine_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from b200attn import ops
    return ops


def listed() -> list[dict]:
    return [
        # one decode step of the ordinary serving batch: launch and latency are everything
        dict(name="append_step", kind="append", batch=32, low=1, high=1, start_low=128, start_high=700, hq=8, hkv=2, dim=256, rot=64,
             axes=1, far=0),
        # newcomers and portions of prompts, ragged
        dict(name="append_ragged", kind="append", batch=32, low=16, high=512, start_low=0, start_high=1000, hq=8, hkv=2, dim=256, rot=64,
             axes=1, far=0),
        # long portions with images: three positions per token, far along a document
        dict(name="append_axes", kind="append", batch=8, low=4096, high=4096, start_low=0, start_high=300, hq=8, hkv=2, dim=256, rot=64,
             axes=3, far=200000),
        # another head layout, every dimension rotated, odd lengths
        dict(name="append_heads", kind="append", batch=13, low=3, high=777, start_low=5, start_high=500, hq=12, hkv=4, dim=128, rot=128,
             axes=1, far=0),
        # the check of four speculated tokens per sequence
        dict(name="chunk_verify", kind="chunk", batch=32, low=4, high=4, start_low=512, start_high=4092, hq=8, hkv=2, dim=256, gate=True,
             singles=False),
        # single tokens over long contexts, few sequences: the cache has to be split to be read by the whole device
        dict(name="chunk_step", kind="chunk", batch=4, low=1, high=1, start_low=30000, start_high=32767, hq=8, hkv=2, dim=256, gate=False,
             singles=False),
        # portions of long prompts behind what earlier portions left
        dict(name="chunk_long", kind="chunk", batch=8, low=2048, high=2048, start_low=2048, start_high=2048, hq=8, hkv=2, dim=256,
             gate=True, singles=False),
        # decoding sequences and portions of prompts in one call, three query heads to a key/value head of 128
        dict(name="chunk_mixed", kind="chunk", batch=24, low=17, high=701, start_low=0, start_high=8000, hq=12, hkv=4, dim=128, gate=False,
             singles=True),
        # one user
        dict(name="sample_one", kind="sample", batch=1, vocab=248320, dtype="float32", spread=2.5, top_k=0, top_p=0.9, min_p=0.0),
        # the ordinary batch, every filter, rows that differ
        dict(name="sample_batch", kind="sample", batch=32, vocab=248320, dtype="float32", spread=2.5, top_k=50, top_p=0.95, min_p=0.05),
        # a full box without a limit on the number of tokens: the flattest rows
        dict(name="sample_full", kind="sample", batch=256, vocab=248320, dtype="float32", spread=2.0, top_k=0, top_p=0.95, min_p=0.0),
        # 16-bit logits with many equal values, an odd vocabulary
        dict(name="sample_odd", kind="sample", batch=48, vocab=65521, dtype="bfloat16", spread=2.5, top_k=40, top_p=1.0, min_p=0.0),
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number between low and high, evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "chunk", "chunk", "sample"])
    if kind == "sample":
        return dict(kind=kind, batch=_spread(rng, 1, 256), vocab=_spread(rng, 1000, 248320), dtype=rng.choice(["float32", "float32", "bfloat16"]),
                    spread=rng.choice([1.5, 2.0, 2.5]), top_k=rng.choice([0, 0, _spread(rng, 1, 1000)]), top_p=rng.choice([1.0, 0.95, 0.8]),
                    min_p=rng.choice([0.0, 0.0, 0.05]))
    batch = _spread(rng, 1, 64)
    hkv, group, dim = rng.choice([(2, 4, 256), (2, 4, 256), (1, 8, 256), (4, 3, 128), (8, 1, 128), (2, 7, 128), (4, 2, 256)])
    heads = dict(hq=hkv * group, hkv=hkv, dim=dim)
    if kind == "append":
        rot = rng.choice([dim, 64, dim // 2])
        high = _spread(rng, 1, max(1, min(4096, 20_000_000 // (hkv * (group + 1) * rot * batch))))
        return dict(kind=kind, batch=batch, low=(high + 1) // rng.choice([2, 8]) or 1, high=high, start_low=0, start_high=_spread(rng, 1, 1000),
                    rot=rot, axes=rng.choice([1, 1, 3]), far=rng.choice([0, 0, 100000]), **heads)
    high = _spread(rng, 1, max(1, min(2048, 8192 // batch)))
    # no more cached bytes and no more products than the largest listed case
    most = min(200_000_000 // (batch * hkv * dim * 4) - high, 300_000_000_000 // (4 * dim * hkv * group * batch * high) - high)
    reach = _spread(rng, 1, max(1, min(32768, most)))
    return dict(kind=kind, batch=batch, low=(high + 1) // rng.choice([2, 8]) or 1, high=high, start_low=reach // 4, start_high=reach,
                gate=rng.random() < 0.5, singles=high > 1 and rng.random() < 0.3, **heads)


# -------------------------------------------------------------------------------------------------------------- lengths
def _lengths(case) -> tuple[list[int], list[int]]:
    """New tokens of every sequence, and the tokens it holds already."""
    rs = np.random.RandomState((case["batch"] * 8191 + case["low"] * 131 + case["high"] * 17 + case["start_high"]) % 2**31)
    new = rs.randint(case["low"], case["high"] + 1, case["batch"])
    held = rs.randint(case["start_low"], case["start_high"] + 1, case["batch"])
    if case.get("singles"):
        new[::2] = 1
    return new.tolist(), held.tolist()


def _visible(case) -> int:
    """(query token, visible key) pairs of one head."""
    return sum(n * h + n * (n + 1) // 2 for n, h in zip(*_lengths(case)))


def work(case) -> dict:
    if case["kind"] == "sample":
        size = 2 if case["dtype"] == "bfloat16" else 4
        # logits read once, one id written; a difference, a scaling, an exponential and a sum for every token
        return dict(bytes=case["batch"] * (case["vocab"] * size + 8 + 20), flops=4 * case["batch"] * case["vocab"])
    new, held = _lengths(case)
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    tokens = sum(new)
    if case["kind"] == "append":
        return dict(bytes=tokens * (2 * (hq + 2 * hkv) * dim * 2 + 8 * case["axes"]), flops=tokens * (hq + hkv) * case["rot"] * 3)
    cached = sum(n + h for n, h in zip(new, held))
    rows = 3 if case["gate"] else 2
    return dict(bytes=cached * hkv * dim * 2 * 2 + tokens * hq * dim * 2 * rows, flops=4 * dim * hq * _visible(case))


# --------------------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=F32).to(BF)


def _table(gen, total: list[int]) -> tuple[torch.Tensor, int]:
    """Page table [batch, most pages] over randomly placed pages, and the pages of the pool."""
    pages = [-(-n // PAGE) for n in total]
    perm = torch.randperm(sum(pages) + 8, generator=gen, device=DEV).to(torch.int32)
    table, at = torch.zeros(len(total), max(pages), dtype=torch.int32, device=DEV), 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[at: at + n]
        at += n
    return table, perm.numel()


def _sample_inputs(case, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    batch, vocab = case["batch"], case["vocab"]
    logits = torch.randn(batch, vocab, generator=gen, device=DEV) * case["spread"]
    # what a trained model is sure of: a few tokens that stand out
    few = max(1, min(24, vocab // 8))
    at = torch.randint(vocab, (batch, few), generator=gen, device=DEV)
    logits.scatter_(1, at, case["spread"] * (3.0 + 3.0 * torch.rand(batch, few, generator=gen, device=DEV)))
    logits = logits.to(getattr(torch, case["dtype"]))
    rs = np.random.RandomState(seed % 2**31)
    low_k, high_k = max(1, case["top_k"] // 2), case["top_k"] + 1
    top_k = rs.randint(low_k, high_k, batch) if case["top_k"] else np.zeros(batch)
    top_p = rs.uniform(case["top_p"] - 0.1, case["top_p"], batch) if case["top_p"] < 1 else np.ones(batch)
    min_p = rs.uniform(0.5 * case["min_p"], case["min_p"], batch)

    def send(a, dtype):
        return torch.from_numpy(np.asarray(a)).to(dtype).to(DEV)
    return dict(kind="sample", logits=logits, uniform=torch.rand(batch, generator=gen, device=DEV),
                temperature=send(rs.uniform(0.6, 1.1, batch), F32), top_k=send(top_k, torch.int32), top_p=send(top_p, F32),
                min_p=send(min_p, F32))


def prepare(case, seed: int) -> dict:
    if case["kind"] == "sample":
        return _sample_inputs(case, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    new, held = _lengths(case)
    hq, hkv, dim, tokens = case["hq"], case["hkv"], case["dim"], sum(new)
    table, pages = _table(gen, [n + h for n, h in zip(new, held)])
    state = dict(kind=case["kind"], new=new, held=held, table=table,
                 cu=torch.tensor([0, *np.cumsum(new).tolist()], dtype=torch.int32, device=DEV),
                 pos=torch.tensor(held, dtype=torch.int64, device=DEV),
                 k_cache=_randn(gen, pages, hkv, PAGE, dim), v_cache=_randn(gen, pages, hkv, PAGE, dim))
    if case["kind"] == "chunk":
        state["q"] = _randn(gen, tokens, hq, dim)
        state["gate"] = _randn(gen, tokens, hq * dim) if case["gate"] else None
        return state
    # normed queries and keys; the values are a part of the projection's rows
    state["q"], state["k"] = _randn(gen, tokens, hq, dim), _randn(gen, tokens, hkv, dim)
    state["v"] = _randn(gen, tokens, (hq + 2 * hkv) * dim)[:, (hq + hkv) * dim:].view(tokens, hkv, dim)
    at = torch.cat([torch.arange(h, h + n) for n, h in zip(new, held)]) + case["far"]
    rot = case["rot"]
    if case["axes"] > 1:
        # patches of 8 x 8 in raster order: time goes on patch by patch, height and width inside one
        inside = torch.cat([torch.arange(n) for n in new])
        state["positions"] = torch.stack([at - inside + inside // 64, at - inside + inside % 64 // 8, at - inside + inside % 8]).to(DEV)
        state["freq_axis"] = (torch.arange(rot // 2, dtype=torch.int32) % 3).to(DEV)
    else:
        state["positions"], state["freq_axis"] = at.to(DEV), None
    state["inv_freq"] = (1.0 / (THETA ** (torch.arange(0, rot, 2, dtype=F32) / rot))).to(DEV)
    return state


# ---------------------------------------------------------------------------------------------------------------- calls
def run(state):
    kind = state["kind"]
    if not own:
        return {"append": _plain_append, "chunk": _plain_chunk, "sample": _plain_sample}[kind](state)
    ops = _ops()
    if kind == "append":
        q = ops.paged_kv_append_rope(state["q"], state["k"], state["v"], state["k_cache"], state["v_cache"], state["table"], state["cu"],
                                     state["pos"], state["positions"], state["inv_freq"], 2 * state["inv_freq"].numel(),
                                     freq_axis=state["freq_axis"])
        return q, state["k_cache"], state["v_cache"]
    if kind == "chunk":
        return ops.paged_gqa_attention_chunk(state["q"], state["k_cache"], state["v_cache"], state["table"], state["cu"], state["pos"],
                                             gate=state["gate"])
    return ops.sample_rows(state["logits"], state["uniform"], state["temperature"], state["top_k"], state["top_p"], state["min_p"])


def _plain_append(state):
    positions, freq = state["positions"], state["inv_freq"]
    if positions.ndim == 2:                     # the axis whose position each frequency takes
        positions = positions[state["freq_axis"].long()].t()
    else:
        positions = positions[:, None]
    angle = positions.to(F64) * freq.to(F64)    # in 64 bits: far positions
    cos, sin = angle.cos().to(F32)[:, None], angle.sin().to(F32)[:, None]
    half = freq.numel()

    def rotate(x):
        x = x.to(F32)
        a, b, rest = x[..., :half], x[..., half: 2 * half], x[..., 2 * half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1).to(BF)
    cu, held, table = state["cu"].long(), state["pos"], state["table"].long()
    tokens = state["q"].shape[0]
    t = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(cu, t, right=True) - 1
    at = held[seq] + t - cu[seq]
    page, slot = table[seq, at // PAGE], at % PAGE
    state["k_cache"][page, :, slot] = rotate(state["k"])
    state["v_cache"][page, :, slot] = state["v"]
    return rotate(state["q"]), state["k_cache"], state["v_cache"]


def _plain_chunk(state):
    q, hkv, dim = state["q"], state["k_cache"].shape[1], state["q"].shape[2]
    tokens, hq = q.shape[:2]
    out, first = torch.empty(tokens, hq * dim, dtype=BF, device=DEV), 0
    for b, (n, h) in enumerate(zip(state["new"], state["held"])):
        pages = state["table"][b, : -(-(n + h) // PAGE)].long()
        k, v = (c[pages].transpose(0, 1).reshape(hkv, -1, dim)[:, : n + h].to(F32) for c in (state["k_cache"], state["v_cache"]))
        rows = q[first: first + n].to(F32).view(n, hkv, hq // hkv, dim).permute(1, 2, 0, 3)       # [hkv, group, n, dim]
        s = rows @ k[:, None].transpose(2, 3) * (1.0 / math.sqrt(dim))
        seen = torch.arange(n + h, device=DEV)[None] <= torch.arange(h, h + n, device=DEV)[:, None]
        s = s.masked_fill(~seen, -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp()
        o = (p @ v[:, None]) / p.sum(-1, keepdim=True)
        o = o.permute(2, 0, 1, 3).reshape(n, hq * dim)
        if state["gate"] is not None:
            o = o / (1.0 + (-state["gate"][first: first + n].to(F32)).exp())
        out[first: first + n] = o.to(BF)
        first += n
    return out


def _plain_sample(state):
    x = state["logits"].to(F64)                 # in 64 bits: long sums, and tokens next to a border
    x = torch.where(x.isnan(), -math.inf, x)
    top, vocab = x.amax(1, keepdim=True), x.shape[1]
    temperature = state["temperature"].to(F64)[:, None]
    w = torch.where(x == top, 1.0, ((x - top) / temperature).exp())
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=DEV)
    k = state["top_k"].long()[:, None]
    keep = (rank < torch.where(k > 0, k, vocab)) & (xs >= top + temperature * state["min_p"].to(F64)[:, None].log())
    ws = ws * keep
    cum = ws.cumsum(1)
    p = state["top_p"].to(F64)[:, None]
    keep &= (cum - ws < p * cum[:, -1:]) | (p >= 1)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    cum = (w * kept).cumsum(1)
    return (cum <= state["uniform"].to(F64)[:, None] * cum[:, -1:]).sum(1)


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed: int):
    state = prepare(case, seed)
    return {"append": _exact_append, "chunk": _exact_chunk, "sample": _exact_sample}[case["kind"]](state)


def _exact_append(state):
    positions, freq = state["positions"].to(F64), state["inv_freq"].to(F64)
    half = freq.numel()
    if positions.ndim == 1:
        angle = torch.outer(positions, freq)
    else:
        angle = torch.stack([positions[int(a)] * f for a, f in zip(state["freq_axis"].tolist(), freq.tolist())], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotated(x):
        y = x.to(F64).clone()
        z = torch.complex(y[..., :half].contiguous(), y[..., half: 2 * half].contiguous()) * turn
        y[..., :half], y[..., half: 2 * half] = z.real, z.imag
        return y
    k, v = rotated(state["k"]), state["v"].to(F64)
    k_cache, v_cache, first = state["k_cache"].to(F64), state["v_cache"].to(F64), 0
    for b, (n, h) in enumerate(zip(state["new"], state["held"])):
        for page in range(h // PAGE, (h + n - 1) // PAGE + 1):
            low, high = max(h, page * PAGE), min(h + n, (page + 1) * PAGE)
            where = int(state["table"][b, page])
            rows = slice(first + low - h, first + high - h)
            k_cache[where, :, low - page * PAGE: high - page * PAGE] = k[rows].transpose(0, 1)
            v_cache[where, :, low - page * PAGE: high - page * PAGE] = v[rows].transpose(0, 1)
        first += n
    return rotated(state["q"]), k_cache, v_cache


def _exact_chunk(state):
    q = state["q"].to(F64)
    hkv, dim = state["k_cache"].shape[1], q.shape[2]
    group = q.shape[1] // hkv
    out, first = [], 0
    for b, (n, h) in enumerate(zip(state["new"], state["held"])):
        pages = state["table"][b, : -(-(n + h) // PAGE)].long()
        hidden = torch.triu(torch.ones(n, n + h, dtype=torch.bool, device=DEV), diagonal=h + 1)
        heads = []
        for g in range(hkv):
            k, v = (c[pages, g].reshape(-1, dim)[: n + h].to(F64) for c in (state["k_cache"], state["v_cache"]))
            for j in range(group):
                s = q[first: first + n, g * group + j] @ k.t() / math.sqrt(dim)
                heads.append(torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v)
        out.append(torch.cat(heads, 1))
        first += n
    out = torch.cat(out)
    return out if state["gate"] is None else out * torch.sigmoid(state["gate"].to(F64))


def _exact_sample(state):
    logits = state["logits"].to(F32).cpu().numpy().astype(np.float64)
    per_row = [state[name].cpu().numpy().astype(np.float64) for name in ("uniform", "temperature", "top_k", "top_p", "min_p")]
    ids = []
    for x, u, t, k, p, m in zip(logits, *per_row):
        weight = np.exp((x - x.max()) / t)
        order = np.argsort(-x, kind="stable")
        count = len(x) if k <= 0 else int(min(k, len(x)))
        best = order[:count]
        best = best[weight[best] >= m]
        if p < 1:
            cum = np.cumsum(weight[best])
            best = best[: int(np.searchsorted(cum, p * cum[-1], side="left")) + 1]
        best = np.sort(best)
        cum = np.cumsum(weight[best])
        ids.append(int(best[min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(best) - 1)]))
    return torch.tensor(ids, dtype=torch.int64, device=DEV)
