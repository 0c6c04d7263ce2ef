"""The operators behind a paged key-value cache: attention of single tokens and chunks of new tokens over pages, the attention weight that every
cached key has received, and the eviction of keys by that weight.

Every case is a plain dict (``op`` names the operator) of sizes that this repository's configurations, tests and benchmark use, or generic
ones.  ``prepare`` builds what a program has in hand before the call, ``run`` makes the call -- the framework's where ``own`` is true,
else the operator's plain form in elementary torch operations.  ``exact`` computes the same outputs from the definition in 64 bits.
"""
from __future__ import annotations

import math
import random
from typing import Any, Dict, List, Tuple

import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------------------------------------
# attn: `singles` sequences bring one token each behind lo .. hi cached ones, and every "rows@cached" of `chunks` is a sequence that brings a chunk.
def _attn(name: str, groups: int, per: int, dim: int, page: int, singles: int = 0, lo: int = 0, hi: int = 0, chunks: str = "", weights: bool = False,
          rope: int = 0, table: str = "fp32") -> Dict[str, Any]:
    return dict(name=name, op="attn", groups=groups, per=per, dim=dim, rope=rope or dim, page=page, singles=singles, lo=lo, hi=hi, chunks=chunks, weights=weights, table=table)


def listed() -> List[Dict[str, Any]]:
    return [
        # one request of a small deployment, a few hundred tokens in: latency
        _attn("decode-1x300", 32, 1, 128, 16, singles=1, lo=300, hi=300),
        # a full batch of requests of unequal lengths, grouped heads: bandwidth
        _attn("decode-gqa-64x16001", 8, 4, 128, 64, singles=64, lo=5, hi=16000),
        # heads of 64, a quarter of them rotated, odd lengths
        _attn("decode-64d-7x1001", 12, 1, 64, 16, singles=7, lo=0, hi=1000, rope=16),
        # the next portion of a long prompt
        _attn("chunk-613@1500", 8, 4, 128, 128, chunks="613@1500"),
        # a whole prompt, as long as the models' contexts
        _attn("prompt-4096", 32, 1, 128, 64, chunks="4096@0"),
        # a step of continuous batching: requests that decode beside the portion of a prompt that fits the step
        _attn("mixed-32+512", 8, 4, 128, 64, singles=32, lo=100, hi=3001, chunks="512@1024"),
        # sixteen requests whose caches will be cut down by weight
        _attn("weights-16x2048", 32, 1, 128, 64, singles=16, lo=2047, hi=2047, weights=True),
        # the portion of a prompt, weights recorded
        _attn("weights-512@2000", 8, 4, 128, 64, chunks="512@2000", weights=True),
        # short prompts and single tokens of a small model together, weights recorded
        _attn("weights-64d-3+5", 12, 1, 64, 32, singles=5, lo=1, hi=700, chunks="37@0 130@55 260@3", weights=True, rope=16, table="bf16"),
        # one request that has outgrown its budget by a page
        dict(name="evict-1x576", op="evict", seqs=1, groups=32, dim=128, page=64, lo=576, hi=576, keep=512, first=4, recent=128),
        # long documents cut down to what a batch of requests may hold
        dict(name="evict-16x8001", op="evict", seqs=16, groups=8, dim=128, page=64, lo=3001, hi=8001, keep=2048, first=4, recent=256),
        # a single very long context of a small model, odd sizes
        dict(name="evict-64d-1x30001", op="evict", seqs=1, groups=12, dim=64, page=16, lo=30001, hi=30001, keep=8191, first=1, recent=1001),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> Dict[str, Any]:
    costs = [work(c) for c in listed()]
    dearest = {k: max(c[k] for c in costs) for k in ("bytes", "flops")}
    while True:
        if rng.random() < 0.75:
            dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128, 256])
            groups, per = rng.choice([1, 2, 4, 8, 8, 12, 32]), rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
            if groups * per > 64:
                continue
            kind = rng.choice(["singles", "chunks", "both"])
            singles = _log(rng, 1, 96) if kind != "chunks" else 0
            lo = rng.choice([0, _log(rng, 1, 16000)])
            hi = max(lo, _log(rng, 1, 16000))
            chunks = " ".join(f"{_log(rng, 2, 4096)}@{rng.choice([0, _log(rng, 1, 12000)])}" for _ in range(rng.choice([1, 1, 2, 5]))) if kind != "singles" else ""
            case = _attn("", groups, per, dim, page, singles, lo if singles else 0, hi if singles else 0, chunks, rng.random() < 0.35, rng.choice([dim, dim, dim // 2, dim // 4]),
                         rng.choice(["fp32", "fp32", "bf16"]))
        else:
            hi = _log(rng, 2, 32000)
            keep = max(1, min(hi - 1, int(hi * rng.uniform(0.05, 0.95))))
            first = min(keep, rng.choice([0, 1, 4, 64]))
            case = dict(op="evict", seqs=_log(rng, 1, 32), groups=rng.choice([1, 2, 4, 8, 12, 32]), dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]),
                        lo=rng.randrange(1, hi + 1), hi=hi, keep=keep, first=first, recent=min(keep - first, int(keep * rng.choice([0.0, 0.1, 0.5, 1.0]))))
        case.pop("name", None)
        cost = work(case)
        if all(cost[k] <= dearest[k] for k in cost):
            return case


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
class _Maker:
    """Tensors from a seed, in the order they are asked for."""

    def __init__(self, seed: int) -> None:
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return torch.empty(shape, device=DEV, dtype=dtype).normal_(0.0, 1.0, generator=self.gen)

    def uniform(self, lo: float, hi: float, *shape: int) -> torch.Tensor:
        return torch.empty(shape, device=DEV, dtype=F32).uniform_(lo, hi, generator=self.gen)


def _spread(lo: int, hi: int, n: int) -> List[int]:
    """n lengths spread evenly from lo to hi."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _steps(case: Dict[str, Any]) -> List[Tuple[int, int]]:
    """(new rows, cached keys) of every sequence of a step."""
    chunks = [tuple(int(v) for v in part.split("@")) for part in case["chunks"].split()]
    return [(1, n) for n in _spread(case["lo"], case["hi"], case["singles"])] + chunks


def _paged(m: _Maker, shuffle: random.Random, lengths: List[int], case: Dict[str, Any]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> page table (sequences, pages of the longest), pages of keys and values.  A sequence's pages lie anywhere in the pool; what is behind its last page is -1."""
    page = case["page"]
    need = [(n + page - 1) // page for n in lengths]
    pool = sum(need) + max(need)
    order = list(range(pool))
    shuffle.shuffle(order)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table.to(DEV), m.normal(pool, case["groups"], page, case["dim"]), m.normal(pool, case["groups"], page, case["dim"])


def _received(m: _Maker, shape: Tuple[int, ...]) -> torch.Tensor:
    """Sums of attention weights: a few keys have much, most have little, some nothing at all."""
    w = (m.uniform(0.0, 1.0, *shape).reciprocal_() * 0.05).clamp_(max=200.0)
    return torch.where(m.uniform(0.0, 1.0, *shape) < 0.1, torch.zeros_like(w), w)


def _prepare_attn(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    m, shuffle = _Maker(seed), random.Random(seed)
    G, per, hs, rope = case["groups"], case["per"], case["dim"], case["rope"]
    steps = _steps(case)
    shuffle.shuffle(steps)
    table, k, v = _paged(m, shuffle, [r + c for r, c in steps], case)
    seqs, row_seq, row_pos = [], [], []
    for i, (rows, cached) in enumerate(steps):
        seqs.append((len(row_seq), rows, cached, i))
        row_seq += [i] * rows
        row_pos += range(cached, cached + rows)
    longest = max(r + c for r, c in steps)
    freq = 10000.0 ** (-torch.arange(0, rope, 2, dtype=F64) / rope)
    angle = torch.outer(torch.arange(longest, dtype=F64), freq).repeat(1, 2)
    kind = TYPES[case["table"]]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    return dict(case=case, qkv=m.normal(len(row_seq), (per + 2) * G * hs), cos=angle.cos().to(DEV, kind), sin=angle.sin().to(DEV, kind), row_pos=i32(row_pos), row_seq=i32(row_seq),
                seqs=i32(seqs), table=table, k=k, v=v, weights=_received(m, k.shape[:3]) if case["weights"] else None, max_rows=max(r for r, _ in steps), max_length=longest,
                host=seqs)


def _prepare_evict(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    m, shuffle = _Maker(seed), random.Random(seed)
    lengths = _spread(case["lo"], case["hi"], case["seqs"])
    shuffle.shuffle(lengths)
    table, k, v = _paged(m, shuffle, lengths, case)
    return dict(case=case, table=table, k=k, v=v, weights=_received(m, k.shape[:3]), lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV), max_length=max(lengths), host=lengths)


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    return (_prepare_attn if case["op"] == "attn" else _prepare_evict)(case, seed)


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state: Dict[str, Any]) -> Any:
    attn = state["case"]["op"] == "attn"
    return ((_own_attn if attn else _own_evict) if own else (_plain_attn if attn else _plain_evict))(state)


def _own_attn(s: Dict[str, Any]) -> Any:
    from lit_gpt_b200 import kernels as K

    c = s["case"]
    out = K.attn_paged(s["qkv"], s["cos"], s["sin"], s["row_pos"], s["row_seq"], s["seqs"], s["table"], s["k"], s["v"], c["groups"] * c["per"], c["groups"], c["dim"], c["rope"],
                       max_rows=s["max_rows"], max_length=s["max_length"], key_weights=s["weights"])
    return (out, s["k"], s["v"]) if s["weights"] is None else (out, s["k"], s["v"], s["weights"])


def _own_evict(s: Dict[str, Any]) -> Any:
    from lit_gpt_b200 import kernels as K

    c = s["case"]
    left = K.evict_paged(s["k"], s["v"], s["weights"], s["table"], s["lengths"], c["keep"], first=c["first"], recent=c["recent"], max_length=s["max_length"])
    return s["k"], s["v"], s["weights"], left


def _turned(x: torch.Tensor, c: torch.Tensor, sn: torch.Tensor, n: int) -> torch.Tensor:
    """The model's rotation of the first n numbers of every head: the two halves of them are the pairs; the result has the type of the keys."""
    a = x[..., :n] if c.dtype == torch.bfloat16 else x[..., :n].to(F32)
    swapped = torch.cat((-a[..., n // 2 :], a[..., : n // 2]), dim=-1)
    return torch.cat((((a * c) + (swapped * sn)).to(x.dtype), x[..., n:]), dim=-1)


def _plain_attn(s: Dict[str, Any]) -> Any:
    case = s["case"]
    G, per, hs, page, n = case["groups"], case["per"], case["dim"], case["page"], case["rope"]
    heads = s["qkv"].view(-1, G, per + 2, hs)
    at = s["row_pos"].long()
    c, sn = s["cos"][at][:, None, None], s["sin"][at][:, None, None]
    q, k_new = _turned(heads[:, :, :per], c, sn, n), _turned(heads[:, :, per : per + 1], c, sn, n)[:, :, 0]
    v_new = heads[:, :, per + 1]
    out = torch.empty(len(at), G, per, hs, dtype=torch.bfloat16, device=DEV)
    for first, rows, cached, t in s["host"]:
        keys = cached + rows
        index = torch.arange(keys, device=DEV)
        where, slot = s["table"][t].long()[index // page], index % page
        mine = slice(first, first + rows)
        s["k"][where[cached:], :, slot[cached:]] = k_new[mine]
        s["v"][where[cached:], :, slot[cached:]] = v_new[mine]
        k, v = s["k"][where, :, slot].to(F32), s["v"][where, :, slot].to(F32)          # (keys, G, hs)
        later = index[None] > index[cached:, None]
        got = torch.zeros(keys, G, device=DEV) if case["weights"] else None
        for g in range(G) if rows > 1 else [slice(0, G)]:                              # (a group at a time where the scores of all take too much room)
            g = slice(g, g + 1) if isinstance(g, int) else g
            scores = torch.einsum("igph,jgh->gpij", q[mine, g].to(F32), k[:, g]) / math.sqrt(hs)
            scores = scores.masked_fill(later, -math.inf)
            w = torch.exp(scores - scores.amax(-1, keepdim=True))
            w = w / w.sum(-1, keepdim=True)
            out[mine, g] = torch.einsum("gpij,jgh->igph", w, v[:, g]).to(torch.bfloat16)
            if got is not None:
                got[:, g] = w.sum(dim=(1, 2)).T
        if got is not None:
            got[:cached] += s["weights"][where[:cached], :, slot[:cached]]
            s["weights"][where, :, slot] = got
    out = out.reshape(len(at), G * per * hs)
    return (out, s["k"], s["v"]) if s["weights"] is None else (out, s["k"], s["v"], s["weights"])


def _plain_evict(s: Dict[str, Any]) -> Any:
    case = s["case"]
    G, page, keep, head, tail = case["groups"], case["page"], case["keep"], case["first"], case["recent"]
    group = torch.arange(G, device=DEV)[:, None]
    for t, n in enumerate(s["host"]):
        if n <= keep:
            continue
        index = torch.arange(n, device=DEV)
        where, slot = s["table"][t].long()[index // page], index % page
        w = s["weights"][where, :, slot].T                                             # (G, n)
        order = torch.sort(w[:, head : n - tail], dim=-1, descending=True, stable=True).indices + head      # equal weights stay in the order of the keys
        kept = torch.cat((index[:head].expand(G, head), order[:, : keep - head - tail], index[n - tail :].expand(G, tail)), dim=1).sort(dim=-1).values
        for x in (s["k"], s["v"], s["weights"]):
            x[where[:keep], group, slot[:keep]] = x[where[kept], group, slot[kept]]
    return s["k"], s["v"], s["weights"], s["lengths"].clamp(max=keep)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------
def work(case: Dict[str, Any]) -> Dict[str, float]:
    G, hs = case["groups"], case["dim"]
    if case["op"] == "attn":
        per, steps = case["per"], _steps(case)
        rows, cached = sum(r for r, _ in steps), sum(c for _, c in steps)
        seen = sum(r * c + r * (r + 1) // 2 for r, c in steps)
        entries = sum(-(-(r + c) // case["page"]) for r, c in steps)
        nbytes = (rows * G * (per + 2) * hs * 2 + 2 * rows * case["rope"] * (4 if case["table"] == "fp32" else 2) + 4 * G * hs * (cached + rows) + rows * G * per * hs * 2
                  + 8 * rows + 16 * len(steps) + 4 * entries + (4 * G * (2 * cached + rows) if case["weights"] else 0))
        return {"bytes": nbytes, "flops": 4 * G * per * hs * seen}
    cut = [n for n in _spread(case["lo"], case["hi"], case["seqs"]) if n > case["keep"]]
    return {"bytes": sum(4 * G * n + G * case["keep"] * (8 * hs + 4) for n in cut) + 8 * case["seqs"], "flops": 0}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------
def exact(case: Dict[str, Any], seed: int) -> Any:
    s = prepare(case, seed)
    return _exact_attn(case, s) if case["op"] == "attn" else _exact_evict(case, s)


def _place(s: Dict[str, Any], t: int, j: int, page: int) -> Tuple[int, int]:
    return s["pages"][t][j // page], j % page


def _exact_attn(case: Dict[str, Any], s: Dict[str, Any]) -> Any:
    G, per, hs, page, n = case["groups"], case["per"], case["dim"], case["page"], case["rope"]
    x = s["qkv"].view(-1, G, per + 2, hs).to(F64)
    cos, sin = (s[name][s["row_pos"].long()].to(F64)[:, None, None] for name in ("cos", "sin"))
    h = x[:, :, : per + 1, :n]
    one, two = h * cos, torch.cat((-h[..., n // 2 :], h[..., : n // 2]), dim=-1) * sin
    if case["table"] == "bf16":            # tables of 16 bits: the model rounds each product as well
        one, two = one.to(torch.bfloat16).to(F64), two.to(torch.bfloat16).to(F64)
    turned = torch.cat(((one + two).to(torch.bfloat16).to(F64), x[:, :, : per + 1, n:]), dim=-1)
    k, v = s["k"].to(F64), s["v"].to(F64)
    a = None if s["weights"] is None else s["weights"].to(F64)
    s["pages"] = s["table"].tolist()
    out = torch.zeros(len(x), G, per, hs, dtype=F64, device=DEV)
    for first, rows, cached, t in s["host"]:
        spots = torch.tensor([_place(s, t, j, page) for j in range(cached + rows)], device=DEV)
        p, o = spots[:, 0], spots[:, 1]
        k[p[cached:], :, o[cached:]], v[p[cached:], :, o[cached:]] = turned[first : first + rows, :, per], x[first : first + rows, :, per + 1]
        if a is not None:
            a[p[cached:], :, o[cached:]] = 0.0
        for g in range(G):
            kg, vg = k[p, g, o], v[p, g, o]
            sums = torch.zeros(cached + rows, dtype=F64, device=DEV)
            for lo in range(0, rows, 512):
                hi = min(lo + 512, rows)
                end = cached + hi
                score = torch.einsum("iph,jh->ipj", turned[first + lo : first + hi, g, :per], kg[:end]) * hs ** -0.5
                seen = torch.arange(end, device=DEV)[None] <= torch.arange(cached + lo, end, device=DEV)[:, None]
                w = torch.softmax(torch.where(seen[:, None], score, -math.inf), dim=-1)
                out[first + lo : first + hi, g] = w @ vg[:end]
                sums[:end] += w.sum(dim=(0, 1))
            if a is not None:
                a[p, g, o] += sums
    out = out.reshape(len(x), -1)
    return (out, k, v) if a is None else (out, k, v, a)


def _exact_evict(case: Dict[str, Any], s: Dict[str, Any]) -> Any:
    page, keep, head, tail = case["page"], case["keep"], case["first"], case["recent"]
    if case["seqs"] * case["groups"] * case["hi"] > 4_000_000:
        return None
    s["pages"] = s["table"].tolist()
    host = s["weights"].cpu()
    for t, n in enumerate(s["host"]):
        if n <= keep:
            continue
        spots = torch.tensor([_place(s, t, j, page) for j in range(n)])
        for g in range(case["groups"]):
            w = host[spots[:, 0], g, spots[:, 1]].tolist()
            ranked = sorted(range(head, n - tail), key=lambda j: (-w[j], j))[: keep - head - tail]
            kept = sorted(ranked + list(range(head)) + list(range(n - tail, n)))
            src, dst = spots[kept].to(DEV), spots[:keep].to(DEV)
            for x in (s["k"], s["v"], s["weights"]):
                x[dst[:, 0], g, dst[:, 1]] = x[src[:, 0], g, src[:, 1]]
    return s["k"], s["v"], s["weights"], torch.tensor([min(n, keep) for n in s["host"]], dtype=torch.int32, device=DEV)
