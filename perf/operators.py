"""The operators behind several answers to one prompt: a decode step of rows that share a prefix, penalties and masks on logits, one draw
per row, and copies of cache slots.

Every case is a plain dict (``op`` names the operator) of sizes that this repository's configurations, tests and benchmark use, or generic
ones.  ``prepare`` builds what a program has in hand before the call, ``run`` makes the call -- the framework's where ``own`` is true,
else the operator's plain form in elementary torch operations.  ``exact`` computes the same outputs from the definition in 64 bits.
"""
from __future__ import annotations

import math
import random
from typing import Any, Dict, List, Optional, Tuple

import numpy as np
import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------------------------------------
def listed() -> List[Dict[str, Any]]:
    return [
        # two answers to a short question, a few tokens in: latency
        dict(name="attn-2x96", op="attn", rows=2, groups=32, per=1, dim=128, rope=128, prefix=96, cap=64, lo=3, hi=3, idle=0, table="fp32"),
        # sixteen answers to an ordinary prompt, one key-value head per query head
        dict(name="attn-16x2048", op="attn", rows=16, groups=32, per=1, dim=128, rope=128, prefix=2048, cap=512, lo=200, hi=200, idle=0, table="fp32"),
        # many answers over a long document, grouped heads, answers of unequal lengths, some of them finished
        dict(name="attn-gqa-64x16001", op="attn", rows=64, groups=8, per=4, dim=128, rope=128, prefix=16001, cap=1024, lo=5, hi=1000, idle=3, table="fp32"),
        # heads of 64 with a quarter of them rotated, odd sizes
        dict(name="attn-64d-7x1001", op="attn", rows=7, groups=12, per=1, dim=64, rope=16, prefix=1001, cap=300, lo=0, hi=299, idle=0, table="fp32"),
        # one row of logits on its way to a sampler of the user's own, repeated tokens penalised
        dict(name="logits-1x32000", op="logits", rows=1, vocab=32000, dtype="bf16", counts=True, bias="", mask=""),
        # a batch under a grammar, with penalties and a bias per request
        dict(name="logits-64x50304", op="logits", rows=64, vocab=50304, dtype="fp32", counts=True, bias="rows", mask="rows"),
        # the draw of a single answer
        dict(name="sample-1x32000", op="sample", rows=1, vocab=32000, dtype="bf16", counts=False, bias="", mask="", top=200, greedy=0),
        # the draw of sixteen answers, repeated tokens penalised
        dict(name="sample-16x32000", op="sample", rows=16, vocab=32000, dtype="bf16", counts=True, bias="", mask="", top=200, greedy=0),
        # a large batch of requests with settings of their own under a grammar, an odd vocabulary
        dict(name="sample-96x50257", op="sample", rows=96, vocab=50257, dtype="fp32", counts=True, bias="one", mask="rows", top=0, greedy=5),
        # one more answer forked from a live request of a small model: states of constant size
        dict(name="slots-fork-1", op="slots", layers=4, slots=4, parts="6x6144xbf16 1x262144xfp32", positional=False, groups=1, copies=1, lo=0, hi=0),
        # sixteen answers forked from one prompt: rings of a window in every layer
        dict(name="slots-fork-15", op="slots", layers=24, slots=24, parts="1024x512xbf16 1024x512xbf16", positional=False, groups=1, copies=15, lo=0, hi=0),
        # a cache by positions compacted: live requests of unequal lengths move to low slots
        dict(name="slots-move-6", op="slots", layers=24, slots=16, parts="4096x576xbf16", positional=True, groups=6, copies=1, lo=37, hi=4001),
    ]


def _parts(text: str) -> List[Tuple[int, int, str]]:
    """What every layer keeps per slot, "positions x numbers x type" each."""
    return [(int(rows), int(cols), t) for rows, cols, t in (part.split("x") for part in text.split())]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> Dict[str, Any]:
    op = rng.choice(["attn", "attn", "attn", "logits", "sample", "sample", "slots"])
    if op == "attn":
        while True:
            dim, groups, per = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8, 12, 32]), rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
            rows, prefix, cap = _log(rng, 1, 128), _log(rng, 1, 20000), _log(rng, 1, 1500)
            # no dearer than sixty-four answers over the long document
            if groups * per * rows * prefix * dim <= 64 * 32 * 16001 * 128 and groups * dim * (prefix + rows * cap) <= 8 * 128 * (16001 + 64 * 1024):
                break
        lo = rng.randrange(cap)
        return dict(op=op, rows=rows, groups=groups, per=per, dim=dim, rope=rng.choice([dim, dim, dim // 2, dim // 4]), prefix=prefix, cap=cap, lo=lo,
                    hi=rng.randrange(lo, cap), idle=rng.choice([0, 0, rows // 5]), table=rng.choice(["fp32", "fp32", "bf16"]))
    if op in ("logits", "sample"):
        case = dict(op=op, rows=_log(rng, 1, 96), vocab=rng.choice([_log(rng, 50, 50304), 32000, 50257, 50304]), dtype=rng.choice(["bf16", "fp32"]),
                    counts=rng.random() < 0.7, bias=rng.choice(["", "one", "rows"]), mask=rng.choice(["", "one", "rows"]))
        if op == "sample":
            case.update(top=rng.choice([0, 1, _log(rng, 2, 500), 200]), greedy=rng.choice([0, 0, case["rows"] // 3]))
        return case
    layers, slots = rng.choice([2, 4, 12, 24]), rng.choice([4, 8, 16, 24])
    positional = rng.random() < 0.5
    if positional:
        parts = rng.choice([f"{_log(rng, 64, 4096)}x576xbf16", f"{_log(rng, 64, 2048)}x512xbf16 1024x256xbf16", f"{_log(rng, 64, 1024)}x129xfp32"])
    else:
        parts = rng.choice([f"3x6144xbf16 1x{_log(rng, 1000, 262144)}xfp32", f"{_log(rng, 64, 1024)}x512xbf16 512x512xbf16", f"{_log(rng, 3, 1000)}x33xbf16"])
    groups = rng.randrange(1, max(2, slots // 4))
    copies = rng.randrange(1, slots // groups)
    rows = min(p[0] for p in _parts(parts))
    lo = rng.randrange(1, rows + 1) if positional else 0
    return dict(op=op, layers=layers, slots=slots, parts=parts, positional=positional, groups=groups, copies=copies, lo=lo,
                hi=rng.randrange(lo, rows + 1) if positional else 0)


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
class _Maker:
    """Tensors from a seed, in the order they are asked for."""

    def __init__(self, seed: int) -> None:
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape: int, std: float = 1.0, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return torch.empty(shape, device=DEV, dtype=dtype).normal_(0.0, std, generator=self.gen)

    def uniform(self, lo: float, hi: float, *shape: int) -> torch.Tensor:
        return torch.empty(shape, device=DEV, dtype=F32).uniform_(lo, hi, generator=self.gen)

    def chance(self, p: float, *shape: int) -> torch.Tensor:
        return self.uniform(0.0, 1.0, *shape) < p


def _spread(lo: int, hi: int, n: int) -> List[int]:
    """n lengths spread evenly from lo to hi."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _own_lengths(case: Dict[str, Any]) -> List[int]:
    """Own tokens before this step of every row that is not idle (-1: idle)."""
    busy = case["rows"] - case["idle"]
    return _spread(case["lo"], case["hi"], busy) + [-1] * case["idle"]


def _prepare_attn(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    m, shuffle = _Maker(seed), random.Random(seed)
    B, G, per, hs, P, cap = case["rows"], case["groups"], case["per"], case["dim"], case["prefix"], case["cap"]
    lens = _own_lengths(case)
    shuffle.shuffle(lens)
    at = torch.arange(P + cap, dtype=F64)
    freq = 10000.0 ** (-torch.arange(0, case["rope"], 2, dtype=F64) / case["rope"])
    angle = torch.outer(at, freq).repeat(1, 2)
    table = TYPES[case["table"]]
    return dict(case=case, qkv=m.normal(B, (per + 2) * G * hs), k_cache=m.normal(B, G, cap, hs), v_cache=m.normal(B, G, cap, hs),
                k_prefix=m.normal(G, P, hs), v_prefix=m.normal(G, P, hs), cos=angle.cos().to(DEV, table), sin=angle.sin().to(DEV, table),
                pos=torch.tensor([P + n if n >= 0 else -1 for n in lens], dtype=torch.int64, device=DEV),
                prefix_len=torch.tensor([P], dtype=torch.int32, device=DEV))


def _prepare_logits(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    m = _Maker(seed)
    B, V = case["rows"], case["vocab"]
    s: Dict[str, Any] = dict(case=case, logits=m.normal(B, V, std=3.0, dtype=F32).to(TYPES[case["dtype"]]), counts=None, bias=None, allowed=None)
    if case["counts"]:   # a few hundred distinct tokens so far, most of them once
        times = (m.uniform(0.0, 1.0, B, V).reciprocal_() * 0.4).clamp_(1.0, 40.0).to(torch.int32)
        s["counts"] = torch.where(m.chance(min(0.5, 300.0 / V), B, V), times, torch.zeros_like(times))
    if case["bias"]:
        shape = (V,) if case["bias"] == "one" else (B, V)
        s["bias"] = torch.where(m.chance(0.02, *shape), m.uniform(-5.0, 5.0, *shape), torch.zeros(shape, device=DEV))
    if case["mask"]:     # a grammar leaves a part of the vocabulary
        shape = (V,) if case["mask"] == "one" else (B, V)
        ok = m.chance(0.3, *shape)
        ok[..., 0] = True
        s["allowed"] = _packed(ok)
    s["repetition"], s["frequency"], s["presence"] = m.uniform(1.0, 1.4, B), m.uniform(0.0, 0.5, B), m.uniform(0.0, 0.5, B)
    if case["op"] == "sample":
        s["temperature"] = m.uniform(0.5, 1.3, B)
        s["temperature"][: case["greedy"]] = 0.0
        s["top_k"] = torch.full((B,), case["top"], dtype=torch.int32, device=DEV)
        s["noise"] = torch.empty(B, V, device=DEV, dtype=F32).exponential_(1.0, generator=m.gen)
    return s


def _packed(ok: torch.Tensor) -> torch.Tensor:
    """Truth values (..., V) as bits: token v is bit v % 32 of word v / 32."""
    V = ok.shape[-1]
    words = torch.zeros((*ok.shape[:-1], (V + 31) // 32 * 32), dtype=torch.int64, device=ok.device)
    words[..., :V] = ok
    words = (words.view(*ok.shape[:-1], -1, 32) << torch.arange(32, device=ok.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _pairs(case: Dict[str, Any], seed: int) -> Tuple[List[int], List[int], List[int]]:
    order = list(range(case["slots"]))
    random.Random(seed).shuffle(order)
    src, dst, lengths = [], [], []
    for g, n in enumerate(_spread(case["lo"], case["hi"], case["groups"])):
        for _ in range(case["copies"]):
            src.append(order[g])
            dst.append(order[case["groups"] + len(dst)])
            lengths.append(n)
    return src, dst, lengths


def _prepare_slots(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    m = _Maker(seed)
    src, dst, lengths = _pairs(case, seed)
    tensors = [m.normal(case["slots"], rows, cols, dtype=TYPES[t]) for _ in range(case["layers"]) for rows, cols, t in _parts(case["parts"])]
    return dict(case=case, tensors=tensors, src=src, dst=dst, lengths=lengths if case["positional"] else None)


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    return {"attn": _prepare_attn, "logits": _prepare_logits, "sample": _prepare_logits, "slots": _prepare_slots}[case["op"]](case, seed)


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state: Dict[str, Any]) -> Any:
    return (_run_own if own else _run_plain)(state)


def _run_own(s: Dict[str, Any]) -> Any:
    from lit_gpt_b200 import kernels as K

    case = s["case"]
    if case["op"] == "attn":
        out = K.attn_decode_shared(s["qkv"], s["cos"], s["sin"], s["pos"], s["k_cache"], s["v_cache"], s["k_prefix"], s["v_prefix"], s["prefix_len"],
                                   case["groups"] * case["per"], case["groups"], case["dim"], case["rope"])
        return out, s["k_cache"], s["v_cache"]
    if case["op"] == "slots":
        K.copy_slots(s["tensors"], s["src"], s["dst"], s["lengths"])
        return s["tensors"]
    how = dict(counts=s["counts"], repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias=s["bias"], allowed=s["allowed"])
    if case["op"] == "logits":
        return K.adjust_logits(s["logits"], **how)
    token, logprob = torch.empty(case["rows"], dtype=torch.int64, device=DEV), torch.empty(case["rows"], dtype=F32, device=DEV)
    K.sample_rows_(s["logits"], token, s["temperature"], s["top_k"], noise=s["noise"], logprob_out=logprob, **how)
    return token, logprob


def _turned(x: torch.Tensor, c: torch.Tensor, sn: torch.Tensor, n: int) -> torch.Tensor:
    """The model's rotation of the first n numbers of every head: the two halves of them are the pairs; the result has the type of the keys."""
    a = x[..., :n] if c.dtype == torch.bfloat16 else x[..., :n].to(F32)
    swapped = torch.cat((-a[..., n // 2 :], a[..., : n // 2]), dim=-1)
    return torch.cat((((a * c) + (swapped * sn)).to(x.dtype), x[..., n:]), dim=-1)


def _plain_attn(s: Dict[str, Any]) -> Any:
    case = s["case"]
    B, G, per, hs, P = case["rows"], case["groups"], case["per"], case["dim"], case["prefix"]
    pos, kc, vc = s["pos"], s["k_cache"], s["v_cache"]
    busy = pos >= 0
    at = pos.clamp(min=0)
    heads = s["qkv"].view(B, G, per + 2, hs)
    c, sn = s["cos"][at][:, None, None], s["sin"][at][:, None, None]
    q, k = _turned(heads[:, :, :per], c, sn, case["rope"]), _turned(heads[:, :, per : per + 1], c, sn, case["rope"])[:, :, 0]
    which, slot = torch.arange(B, device=DEV), (at - P).clamp(min=0)
    kc[which, :, slot] = torch.where(busy[:, None, None], k, kc[which, :, slot])
    vc[which, :, slot] = torch.where(busy[:, None, None], heads[:, :, per + 1], vc[which, :, slot])
    q = q.to(F32)
    shared = torch.einsum("bgph,gjh->bgpj", q, s["k_prefix"].to(F32))
    mine = torch.einsum("bgph,bgjh->bgpj", q, kc.to(F32))
    mine = mine.masked_fill((torch.arange(kc.shape[2], device=DEV)[None] > slot[:, None])[:, None, None], -math.inf)
    scores = torch.cat((shared, mine), dim=-1) / math.sqrt(hs)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    seen = (torch.arange(kc.shape[2], device=DEV)[None] <= slot[:, None])[:, None, :, None]
    out = torch.einsum("bgpj,gjh->bgph", w[..., :P], s["v_prefix"].to(F32)) + torch.einsum("bgpj,bgjh->bgph", w[..., P:], torch.where(seen, vc.to(F32), 0.0))
    out = torch.where(busy[:, None, None, None], out, 0.0)
    return out.reshape(B, G * per * hs).to(torch.bfloat16), kc, vc


def _plain_adjusted(s: Dict[str, Any]) -> torch.Tensor:
    l = s["logits"].to(F32)
    V = l.shape[1]
    if s["counts"] is not None:
        n = s["counts"].clamp(min=0).to(F32)
        r, f, p = s["repetition"][:, None], s["frequency"][:, None], s["presence"][:, None]
        pulled = torch.where(l > 0, l / r, l * r)
        l = torch.where(n > 0, (pulled - f * n) - p, l)
    if s["bias"] is not None:
        l = l + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEV)
        l = torch.where(((s["allowed"][..., v // 32] >> (v % 32)) & 1) != 0, l, -math.inf)
    return l


def _plain_sample(s: Dict[str, Any]) -> Any:
    l = _plain_adjusted(s)
    B, V = l.shape
    T, k = s["temperature"][:, None].to(F64), s["top_k"][:, None]
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices      # equal logits stay in the order of the tokens
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=DEV).expand(B, V))
    kept = ((rank < torch.where(k > 0, k, V)) | (T <= 0)) & (l > -math.inf)
    top = l.amax(-1, keepdim=True)
    weight = torch.where(kept, (l.to(F64) - top) / torch.where(T > 0, T, 1.0), -math.inf)
    score = torch.where(T > 0, weight - torch.log(s["noise"].to(F64)), weight)
    best = score == score.amax(-1, keepdim=True)
    token = torch.where(best, torch.arange(V, device=DEV), V).amin(-1)
    logprob = weight.gather(1, token[:, None])[:, 0] - torch.log(torch.exp(weight).sum(-1))
    return token, logprob.to(F32)


def _run_plain(s: Dict[str, Any]) -> Any:
    op = s["case"]["op"]
    if op == "attn":
        return _plain_attn(s)
    if op == "logits":
        return _plain_adjusted(s)
    if op == "sample":
        return _plain_sample(s)
    src, dst = torch.tensor(s["src"], device=DEV), torch.tensor(s["dst"], device=DEV)
    for t in s["tensors"]:
        if s["lengths"] is None:
            t[dst] = t[src]
        else:
            for a, b, n in zip(s["src"], s["dst"], s["lengths"]):
                t[b, :n] = t[a, :n]
    return s["tensors"]


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------
def work(case: Dict[str, Any]) -> Dict[str, float]:
    if case["op"] == "attn":
        B, G, per, hs, P = case["rows"], case["groups"], case["per"], case["dim"], case["prefix"]
        before = [n for n in _own_lengths(case) if n >= 0]
        keys = P * len(before) + sum(n + 1 for n in before)
        table = 4 if case["table"] == "fp32" else 2
        nbytes = (len(before) * G * (per + 2) * hs * 2 + 2 * len(before) * case["rope"] * table + 4 * G * hs * (P + sum(before)) + 4 * len(before) * G * hs
                  + B * G * per * hs * 2 + 8 * B)
        return {"bytes": nbytes, "flops": 4 * G * per * hs * keys}
    if case["op"] in ("logits", "sample"):
        B, V = case["rows"], case["vocab"]
        a_row = V * (2 if case["dtype"] == "bf16" else 4) + (4 * V if case["counts"] else 0) + (4 * V if case["bias"] == "rows" else 0) + (V // 8 if case["mask"] == "rows" else 0)
        nbytes = B * a_row + (4 * V if case["bias"] == "one" else 0) + (V // 8 if case["mask"] == "one" else 0)
        if case["op"] == "logits":
            return {"bytes": nbytes + 4 * B * V, "flops": 8 * B * V}
        return {"bytes": nbytes + 4 * (B - case["greedy"]) * V + 12 * B, "flops": 12 * B * V}
    _, _, lengths = _pairs(case, 0)
    once = 0
    for rows, cols, t in _parts(case["parts"]):
        each = cols * (2 if t == "bf16" else 4)
        once += sum((n if case["positional"] else rows) * each for n in lengths[:: case["copies"]])
    return {"bytes": case["layers"] * once * (1 + case["copies"]), "flops": 0}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------
def exact(case: Dict[str, Any], seed: int) -> Any:
    s = prepare(case, seed)
    if case["op"] == "slots":
        for t in s["tensors"]:
            for i, (a, b) in enumerate(zip(s["src"], s["dst"])):
                n = t.shape[1] if s["lengths"] is None else s["lengths"][i]
                t[b].narrow(0, 0, n).copy_(t[a].narrow(0, 0, n))
        return s["tensors"]
    if case["op"] == "attn":
        return _exact_attn(case, s)
    return _exact_logits(case, s)


def _exact_attn(case: Dict[str, Any], s: Dict[str, Any]) -> Any:
    B, G, per, hs, P, n = case["rows"], case["groups"], case["per"], case["dim"], case["prefix"], case["rope"]
    if G * per * B * (P + case["hi"]) > 1.2e9:
        return None
    kc, vc = s["k_cache"].to(F64), s["v_cache"].to(F64)
    out = torch.zeros(B, G, per, hs, dtype=F64, device=DEV)
    positions = s["pos"].tolist()
    x = s["qkv"].view(B, G, per + 2, hs).to(F64)
    step = torch.bfloat16 if case["table"] == "bf16" else None      # tables of 16 bits: the model rounds each product as well
    for b, p in enumerate(positions):
        if p < 0:
            continue
        c, sn = s["cos"][p].to(F64), s["sin"][p].to(F64)
        h = x[b, :, : per + 1, :n]
        other = torch.cat((-h[..., n // 2 :], h[..., : n // 2]), dim=-1)
        one, two = h * c, other * sn
        if step is not None:
            one, two = one.to(step).to(F64), two.to(step).to(F64)
        turned = torch.cat(((one + two).to(torch.bfloat16).to(F64), x[b, :, : per + 1, n:]), dim=-1)
        i = p - P
        kc[b, :, i], vc[b, :, i] = turned[:, per], x[b, :, per + 1]
        for g in range(G):
            keys = torch.cat((s["k_prefix"][g].to(F64), kc[b, g, : i + 1]))
            values = torch.cat((s["v_prefix"][g].to(F64), vc[b, g, : i + 1]))
            out[b, g] = torch.softmax(turned[g, :per] @ keys.T * hs ** -0.5, dim=-1) @ values
    return out.reshape(B, -1), kc, vc


def _exact_logits(case: Dict[str, Any], s: Dict[str, Any]) -> Any:
    B, V = case["rows"], case["vocab"]
    host = {k: v.float().cpu().numpy() if torch.is_tensor(v) and v.dtype == torch.bfloat16 else v.cpu().numpy() if torch.is_tensor(v) else v for k, v in s.items()}
    # the draw compares adjusted logits as the 32-bit numbers that they are, so that equal ones stay equal; the logits themselves come in 64 bits
    kind = np.float64 if case["op"] == "logits" else np.float32
    l = host["logits"].astype(kind)
    if case["counts"]:
        n = host["counts"].astype(kind)
        r, f, p = (host[k].astype(kind).reshape(B, 1) for k in ("repetition", "frequency", "presence"))
        with np.errstate(all="ignore"):
            less = np.where(l > 0, l / r, l * r) - f * n
        l = np.where(n > 0, less - p, l)
    if case["bias"]:
        l = l + host["bias"].astype(kind)
    if case["mask"]:
        words = host["allowed"].view(np.uint32).reshape(-1, host["allowed"].shape[-1])
        bits = np.unpackbits(np.ascontiguousarray(words).view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
        l = np.where(bits, l, kind(-np.inf))
    if case["op"] == "logits":
        return torch.from_numpy(np.ascontiguousarray(l)).to(DEV)
    out, prob = np.zeros(B, dtype=np.int64), np.zeros(B)
    for b in range(B):
        row, T, k = l[b].astype(np.float64), float(host["temperature"][b]), int(host["top_k"][b])
        order = np.argsort(-row, kind="stable")[: k if k > 0 and T > 0 else V]
        order = order[row[order] > -np.inf]
        weight = (row[order] - row[order[0]]) / (T if T > 0 else 1.0)
        score = weight - np.log(host["noise"][b][order].astype(np.float64)) if T > 0 else weight
        at = np.flatnonzero(score == score.max())
        at = at[np.argmin(order[at])]
        out[b], prob[b] = order[at], weight[at] - np.log(np.exp(weight).sum())
    return torch.from_numpy(out).to(DEV), torch.from_numpy(prob).to(DEV)
