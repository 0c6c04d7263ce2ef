"""Steps over a paged cache and its eviction, restated on the CPU: what csrc/paged_attn.cu and csrc/paged_evict.cu compute, in 64 bits."""
import math
import random

import torch

F64 = torch.float64


def make(steps, groups, per, hs, page, rope=None, table=torch.float32, seed=0, spare=2, weights=True, idle=()):
    """steps: per sequence (new rows, cached keys).  Pages lie anywhere in the pool, the sequences' rows of the page table in another order than the sequences."""
    g, r = torch.Generator().manual_seed(seed), random.Random(seed)
    rope = hs if rope is None else rope
    n = sum(rows for rows, _ in steps)
    longest = max(max(rows + cached for rows, cached in steps), 1)
    need = [-(-(rows + cached) // page) for rows, cached in steps]
    pool = sum(need) + spare
    order = list(range(pool))
    r.shuffle(order)
    where = list(range(len(steps)))
    r.shuffle(where)
    pages = torch.full((len(steps), -(-longest // page) + 1), -1, dtype=torch.int32)
    seqs, row_seq, row_pos = [], [], []
    for i, (rows, cached) in enumerate(steps):
        pages[where[i], : need[i]] = torch.tensor([order.pop() for _ in range(need[i])], dtype=torch.int32)
        seqs.append((len(row_seq), rows, cached, where[i]))
        row_seq += [i] * rows
        row_pos += range(cached, cached + rows)
    angle = torch.outer(torch.arange(longest, dtype=F64), 10000.0 ** (-torch.arange(0, max(rope, 1), 2, dtype=F64)[: rope // 2] / max(rope, 1))).repeat(1, 2)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return dict(qkv=rnd(n, (per + 2) * groups * hs), cos=angle.cos().to(table), sin=angle.sin().to(table), row_pos=i32(row_pos), row_seq=i32(row_seq), seqs=i32(seqs), pages=pages,
                k=rnd(pool, groups, page, hs), v=rnd(pool, groups, page, hs), kw=torch.rand(pool, groups, page, generator=g) * 3 if weights else None, groups=groups, per=per, hs=hs,
                rope=rope, max_rows=max(max(rows for rows, _ in steps), 1), max_length=longest)


def turn(x, c, s, n):
    """apply_rope with the model's rounding points."""
    a = x[..., :n] if c.dtype == torch.bfloat16 else x[..., :n].float()
    other = torch.cat((-a[..., n // 2 :], a[..., : n // 2]), -1)
    return torch.cat(((a * c + other * s).bfloat16(), x[..., n:]), -1)


def step(d, rounded=0.0):
    """-> result, bound of its error beside the final rounding, keys, values, key weights and the bound of their error.

    A result's bound: weights that are off by a factor 1 +- off make 2 off sum_j w_j |v_j|, with off the sum of
      * the error of a score: hs + 2 roundings of 2^-24 of sum |q k| / sqrt(hs), in the exponent and once more in the row's maximum;
      * the rounding of the exponent's argument, 2^-23 of the largest score's distance (at most 2 max |s|), and of ex2, 2^-22;
      * a probability in two bf16 numbers: 2^-16 -- or in one: `rounded`, 2^-8 (of that the sums know nothing: once and not twice);
      * sums of n products in fp32: (n + 64) 2^-24, n keys at most.
    A key's weight: the same without the probability's rounding (the sums of exponentials are of unrounded ones), of the step's part, and a rounding of 2^-24 for every one of its
    additions."""
    G, per, hs, page = d["groups"], d["per"], d["hs"], d["k"].shape[2]
    n = d["qkv"].shape[0]
    heads = d["qkv"].view(n, G, per + 2, hs)
    out, slack = torch.zeros(n, G, per, hs, dtype=F64), torch.zeros(n, G, per, hs, dtype=F64)
    k, v = d["k"].clone(), d["v"].clone()
    kw = None if d["kw"] is None else d["kw"].to(F64)
    kw_slack = None if kw is None else torch.zeros_like(kw)
    for i, (first, rows, cached, at) in enumerate(d["seqs"].tolist()):
        if rows <= 0:
            continue
        total = min(cached + rows, d["max_length"])
        place = []
        for j in range(total):
            id_ = int(d["pages"][at, j // page]) if j // page < d["pages"].shape[1] else -1
            place.append((id_, j % page) if 0 <= id_ < len(k) else None)
        turned = {}
        mine = [int(x) == i for x in d["row_seq"][first : first + rows]]   # (a row of no sequence, or of another: no query, and no key in its place)
        for r in range(rows):
            row = first + r
            if not mine[r]:
                if cached + r < total:
                    place[cached + r] = None
                continue
            p = int(d["row_pos"][row])
            c, s = d["cos"][p], d["sin"][p]
            turned[r] = turn(heads[row, :, : per + 1], c, s, d["rope"])
            j = cached + r
            if j < total and place[j] is not None:
                id_, o = place[j]
                k[id_, :, o], v[id_, :, o] = turned[r][:, per], heads[row, :, per + 1]
                if kw is not None:
                    kw[id_, :, o] = 0.0
        there = [j for j in range(total) if place[j] is not None]
        if not there:
            continue
        ids, os_ = torch.tensor([place[j][0] for j in there]), torch.tensor([place[j][1] for j in there])
        keys, values = k[ids, :, os_].to(F64).transpose(0, 1), v[ids, :, os_].to(F64).transpose(0, 1)
        index = torch.tensor(there)
        got, err = torch.zeros(G, len(there), dtype=F64), torch.zeros(G, len(there), dtype=F64)
        for r in range(rows):
            seen = index <= cached + r
            if not seen.any() or not mine[r]:
                continue
            q = turned[r][:, :per].to(F64)
            ks, vs = keys[:, seen], values[:, seen]
            score = q @ ks.transpose(1, 2) / math.sqrt(hs)
            w = torch.softmax(score, -1)
            out[first + r] = w @ vs
            size = (q.abs() @ ks.abs().transpose(1, 2)).amax() / math.sqrt(hs)
            off = 2 * (hs + 2) * 2 ** -24 * size + 2 ** -23 * 2 * score.abs().amax() + 2 ** -22 + (ks.shape[1] + 64) * 2 ** -24
            slack[first + r] = (2 * off + max(rounded, 2 ** -15)) * (w @ vs.abs())
            got[:, seen] += w.sum(1)
            err[:, seen] += 2 * off * w.sum(1)
        if kw is not None:
            before = kw[ids, :, os_].T
            kw[ids, :, os_] = (before + got).T
            kw_slack[ids, :, os_] = (err + (rows * per + 8) * 2 ** -24 * (before + got)).T
    return out.reshape(n, -1), slack.reshape(n, -1), k, v, kw, kw_slack


def evict(k, v, kw, pages, lengths, keep, first=0, recent=0, rows=None):
    """-> keys, values, weights, lengths behind the call."""
    k, v, kw, left = k.clone(), v.clone(), kw.clone(), list(lengths)
    page, pool = k.shape[2], k.shape[0]
    for i, n in enumerate(lengths):
        at = i if rows is None else rows[i]
        if n <= keep:
            continue
        ids = pages[at, : -(-n // page)].tolist()
        if any(not 0 <= x < pool for x in ids):
            continue
        spot = [(ids[j // page], j % page) for j in range(n)]
        for g in range(k.shape[1]):
            w = [kw[a, g, b].item() for a, b in spot]
            rank = sorted(range(first, n - recent), key=lambda j: (-(math.inf if w[j] != w[j] else w[j]), w[j] == w[j], j))[: keep - first - recent]
            kept = sorted(list(range(first)) + rank + list(range(n - recent, n)))
            for x in (k, v, kw):
                moved = [x[spot[j][0], g, spot[j][1]].clone() for j in kept]
                for j, m in enumerate(moved):
                    x[spot[j][0], g, spot[j][1]] = m
        left[i] = keep
    return k, v, kw, left
