"""Steps over a paged cache where kernels have to agree on what they hold and whose rows they are: wide groups, few single tokens, rows that are masked out, numbers that are not finite.
Against the formulas in 64 bits (paged_oracle.py, which derives the tolerances)."""
import pytest
import torch

import paged_oracle as oracle
from paged_oracle import F64, make
from test_gpu_paged import E, K, call, check, formula, launch, on_gpu, path, same  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("per,hs", [(17, 64), (20, 128), (32, 64), (33, 128), (48, 128), (71, 64), (128, 64), (129, 128)])
def test_single_tokens_of_wide_groups(K, formula, weights, per, hs):
    for cached in ([300], [4100] * (16 if per <= 32 else 4), [5, 0, 2000]):   # (wider ones go to the tensor memory however few the keys are)
        d = make([(1, n) for n in cached], 1, per, hs, 64, weights=weights, seed=per)
        check(call(K, d), formula(d))


@pytest.mark.parametrize("tune,per,rows,n", [(1, 4, 100, 40), (3, 4, 100, 40), (0, 130, 9, 60), (1, 1, 4096, 200)])
@pytest.mark.parametrize("weights", [False, True])
def test_sequences_that_share_rows(E, tune, per, rows, n, weights):
    """More items than the step's rows can come to: none is done, and nothing is read of results that nobody left."""
    G, hs = 2, 64
    d = make([(rows, 20)], G, per, hs, 16, weights=weights, seed=rows)
    first = d["seqs"][0].tolist()
    d["seqs"] = torch.tensor([first] * n, dtype=torch.int32)
    d["row_seq"] = torch.arange(rows, dtype=torch.int32) % n
    d["max_rows"] = rows
    ref = oracle.step({**d, "seqs": d["seqs"][:1], "row_seq": torch.zeros(rows, dtype=torch.int32)})   # (for the pages)
    before = E.attn_paged_tune(tune)
    try:
        junk = torch.full((1 << 26,), float("nan"), device="cuda")   # what a workspace may find in its place
        del junk
        out, k, v, kw = call(E, d)
    finally:
        E.attn_paged_tune(before)
    assert not out.any() and same(k.cpu(), ref[2]) and same(v.cpu(), ref[3])
    if weights:
        at = d["pages"][first[3]]
        want = d["kw"].clone()
        for j in range(20, 20 + rows):
            want[at[j // 16], :, j % 16] = 0.0
        assert same(kw.cpu(), want)


@pytest.mark.parametrize("weights", [False, True])
def test_sequences_that_share_rows_on_the_tensor_memory(E, weights):
    rows, n, G, hs, length = 4096, 4096, 32, 64, 100000
    r = torch.Generator(device="cuda").manual_seed(1)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    qkv = torch.randn(rows, 3 * G * hs, device="cuda", generator=r).bfloat16()
    table = torch.full((1, 391), -1, dtype=torch.int32, device="cuda")
    k, v = (torch.ones(2, G, 256, hs, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kw = torch.ones(2, G, 256, device="cuda") if weights else None
    cos, sin = torch.ones(rows, hs, device="cuda"), torch.zeros(rows, hs, device="cuda")
    junk = torch.full((1 << 27,), float("nan"), device="cuda")
    del junk
    out = E.attn_paged(qkv, cos, sin, torch.arange(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"), i32(0, rows, length - rows, 0).expand(n, 4).contiguous(),
                       table, k, v, G, G, hs, hs, max_rows=rows, max_length=length, key_weights=kw)
    assert not out.any() and (k == 1).all() and (v == 1).all() and (kw is None or (kw == 1).all())


def check_with_nan(got, bad, clean):
    """What the formula of the spoilt inputs says is NaN is; everything else is what it is without them."""
    out, kw = got[0].cpu().to(F64), None if got[3] is None else got[3].cpu().to(F64)
    wrong = torch.isnan(bad[0])
    assert wrong.any() and torch.equal(torch.isnan(out), wrong)
    over = ((out - clean[0]).abs() - (2 ** -8 * clean[0].abs() + clean[1]))[~wrong]
    assert over.numel() == 0 or over.max().item() <= 0, over.max().item()
    if kw is not None:
        wrong = torch.isnan(bad[4])
        assert wrong.any() and torch.equal(torch.isnan(kw), wrong)
        over = ((kw - clean[4]).abs() - clean[5])[~wrong]
        assert over.max().item() <= 0, over.max().item()


def one_of_nan(K, formula, weights, steps, where, hs, groups, per, page):
    d = make(steps, groups, per, hs, page, rope=0 if where == "infinite query" else None, weights=weights, seed=len(steps) + per)
    s = len(steps) // 2
    first, rows, cached, at = d["seqs"][s].tolist()
    g = groups - 1
    row = (first + rows // 2, g, per - 1, 3)
    heads = lambda of: of["qkv"].view(-1, groups, per + 2, hs)
    if where == "infinite query":                    # scores of +inf
        d["k"][..., 3] = heads(d)[:, :, per, 3] = 1.0
    clean = formula(d)
    spoilt = {k: v.clone() if torch.is_tensor(v) else v for k, v in d.items()}
    if where == "key" and cached > 0:                # an older one
        j = cached * 2 // 3
        spoilt["k"][d["pages"][at, j // page], g, j % page, 5] = float("nan")
    elif where == "key":                             # the step's own
        heads(spoilt)[first + rows // 2, g, per, hs - 1] = float("nan")
    else:
        heads(spoilt)[row] = float("nan" if where == "query" else "inf")
    check_with_nan(call(K, spoilt), formula(spoilt), clean)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("steps", [[(1, 0)], [(1, 300)], [(1, 40), (1, 700), (1, 9)], [(1, 5000)], [(1, 40), (5, 3), (1, 9)], [(200, 100)], [(1, 60), (130, 700), (3, 0)]],
                         ids=["first", "token", "tokens", "long", "short chunk", "chunk", "mixed"])
def test_what_is_not_a_number_stays_so(K, formula, weights, steps):
    """A query that holds NaN, a key that does: results of the heads that see it are NaN, and so is the weight of every key that they see; no other's."""
    for where in ("query", "key", "infinite query"):
        for hs, groups, per, page in ((64, 2, 4, 16), (128, 3, 1, 64), (128, 1, 16, 32)):
            one_of_nan(K, formula, weights, steps, where, hs, groups, per, page)


def poison():
    """What a workspace may find in its place."""
    junk = [torch.full((1 << n,), float("nan"), device="cuda") for n in range(7, 27) for _ in range(2)]
    del junk


def one_of_strangers(K, formula, weights, steps, which, hs, groups, per, page):
    d = make(steps, groups, per, hs, page, weights=weights, seed=len(steps) + per)
    n = len(d["row_seq"])
    for s, (first, rows, cached, at) in enumerate(d["seqs"].tolist()):
        if s % 3 == 1 and which != "all":
            continue
        out = {"the end": range(rows - max(rows // 3, 1), rows), "the beginning": range(max(rows // 3, 1)), "every third": range(0, rows, 3), "all": range(rows), "another's": range(rows // 2, rows)}[which]
        for r in out:
            d["row_seq"][first + r] = (s + 1) % len(steps) if which == "another's" and len(steps) > 1 else (-1, len(steps), -(2 ** 31), 2 ** 31 - 1)[r % 4]
            j = cached + r
            d["k"][d["pages"][at, j // page], :, j % page], d["v"][d["pages"][at, j // page], :, j % page] = float("nan"), float("inf")
    want = formula(d)
    poison()
    t = on_gpu(d)
    got = launch(K, t), t["k"], t["v"], t["kw"]
    check(got, want)
    for row in range(n):
        s = int(d["row_seq"][row])
        if not 0 <= s < len(steps) or not d["seqs"][s, 0] <= row < d["seqs"][s, 0] + d["seqs"][s, 1]:
            assert not got[0][row].any()
    poison()
    t = on_gpu(d)
    assert same(got[0], launch(K, t)) and (not weights or same(got[3], t["kw"]))


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("steps", [[(1, 0), (1, 40), (1, 70)], [(1, 300)], [(40, 25)], [(5, 0), (7, 90), (3, 31), (8, 2)], [(300, 200)], [(1, 60), (170, 333), (2, 0), (90, 7)]],
                         ids=["tokens", "token", "prompt", "short chunks", "chunk", "mixed"])
def test_rows_within_a_range_that_are_not_the_sequence_s(K, formula, weights, steps):
    """They have no query and no key, whatever lies in their places: results of zero, weights and pages as they were, nothing of them in the other rows."""
    layouts = ((64, 2, 4, 16), (128, 3, 1, 64), (128, 1, 20, 32), (64, 1, 130, 256))
    for i, which in enumerate(("the end", "the beginning", "every third", "all", "another's")):
        for layout in (layouts[i % 4], layouts[(i + 1) % 4]):
            one_of_strangers(K, formula, weights, steps, which, *layout)


# ---- single tokens without weights, every sequence and group by a cluster in one launch -------------------------------------------------
TOKENS = [(1, 0), (1, 31), (1, 300), (1, 64)]


@pytest.fixture
def one_launch(E):
    before = E.attn_paged_tune(4)
    yield lambda d, **kw: call(E, d, **kw)
    E.attn_paged_tune(before)


def tokens(groups=2, per=4, hs=128, page=32, **kw):
    d = make(TOKENS, groups, per, hs, page, weights=False, **kw)
    assert d["max_rows"] == 1
    return d


def test_one_launch_rotations(one_launch):
    for table in (torch.float32, torch.bfloat16):
        for rope in (0, 2, 16, 48, 64):
            d = tokens(hs=64, rope=rope, table=table, seed=rope)
            check(one_launch(d), oracle.step(d))


def test_one_launch_positions_apart_from_places(one_launch):
    d = tokens(seed=9)
    d["cos"], d["sin"] = (torch.cat([t] * 3) for t in (d["cos"], d["sin"]))
    d["row_pos"] = (d["row_pos"].long() * 7 + 3) % len(d["cos"])
    want = oracle.step(d)
    check(one_launch(d), want)
    d["cos"], d["sin"] = d["cos"][d["row_pos"]], d["sin"][d["row_pos"]]
    check(one_launch(d, table_preselected=True), want)
    d["qkv"] = d["qkv"].view(2, 2, -1)                       # leading dimensions
    check(one_launch(d, table_preselected=True), want)


def test_one_launch_strided_rows_and_a_wider_page_table(E, one_launch):
    d = tokens(seed=10)
    want = oracle.step(d)
    t = on_gpu(d)
    n, width = d["qkv"].shape
    wide = torch.zeros(n, width + 72, device="cuda", dtype=torch.bfloat16)
    wide[:, :width] = t["qkv"]
    apart = torch.full((len(d["pages"]), 50), 77, device="cuda", dtype=torch.int32)
    apart[:, : d["pages"].shape[1]] = t["pages"]
    t["qkv"], t["pages"] = wide[:, :width], apart[:, : d["pages"].shape[1]]
    check((launch(E, t), t["k"], t["v"], t["kw"]), want)


@pytest.mark.parametrize("layout", ["keys beside values", "group by group", "apart"])
def test_one_launch_page_layouts(E, one_launch, layout):
    d = tokens(groups=3, per=2, seed=12)
    t = on_gpu(d)
    P, G, page, hs = d["k"].shape
    if layout == "keys beside values":
        both = torch.empty(P, 2, G, page, hs, device="cuda", dtype=torch.bfloat16)
        k, v = both[:, 0], both[:, 1]
    elif layout == "group by group":
        k, v = (torch.empty(G, P, page, hs, device="cuda", dtype=torch.bfloat16).transpose(0, 1) for _ in range(2))
    else:
        k, v = (torch.empty(P * (G * (page * hs + 8) + 64), device="cuda", dtype=torch.bfloat16).as_strided((P, G, page, hs), (G * (page * hs + 8) + 64, page * hs + 8, hs, 1)) for _ in range(2))
    k.copy_(t["k"])
    v.copy_(t["v"])
    t["k"], t["v"] = k, v
    check((launch(E, t), k.contiguous(), v.contiguous(), None), oracle.step(d))


def test_one_launch_offsets_past_32_bits(E, one_launch):
    d = tokens(groups=1, per=2, page=256, seed=13)
    t = on_gpu(d)
    P, far = len(d["k"]), 2 ** 31 // (256 * 128) + 5
    k, v = (torch.empty(far + P, 1, 256, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    k[far:], v[far:] = t["k"], t["v"]
    t.update(k=k, v=v, pages=torch.where(t["pages"] >= 0, t["pages"] + far, -1).int())
    check((launch(E, t), k[far:], v[far:], None), oracle.step(d))


def test_one_launch_reads_nothing_behind_the_last_key(one_launch):
    d = tokens(seed=14)
    page, want = d["k"].shape[2], oracle.step(d)
    used = torch.zeros(d["k"].shape[0], page, dtype=torch.bool)
    for first, rows, cached, at in d["seqs"].tolist():
        for j in range(cached + rows):
            used[d["pages"][at, j // page], j % page] = True
    for x, bad in ((d["k"], float("nan")), (d["v"], float("inf"))):
        x.permute(0, 2, 1, 3)[~used] = bad
    check(one_launch(d), (*want[:2], *oracle.step(d)[2:]))


def test_one_launch_bounds_and_sequences_that_do_not_fit(one_launch):
    d = tokens(seed=15)
    d["max_length"] = 60                                     # keys from here on are dropped: the new ones of the two longest among them
    check(one_launch(d), oracle.step(d))
    for seq in ((2, 1, 300, 99), (2, 1, 300, -1), (4, 1, 0, 0), (-1, 1, 0, 0), (2, 2, 300, 0), (2, 1, -3, 0)):
        d = tokens(seed=15)
        want = oracle.step({**d, "seqs": torch.cat((d["seqs"][:2], torch.zeros(1, 4, dtype=torch.int32), d["seqs"][3:]))})
        d["seqs"][2] = torch.tensor(seq, dtype=torch.int32)
        got = one_launch(d)
        check(got, want)
        assert not got[0][2].any()


def test_one_launch_same_bits_two_streams_and_graphs(E, one_launch):
    ds = [tokens(seed=20), tokens(hs=64, per=16, seed=21)]
    wants, ts = [oracle.step(d) for d in ds], [on_gpu(d) for d in ds]
    first = [launch(E, t) for t in ts]
    for _ in range(3):
        assert all(same(a, launch(E, t)) for a, t in zip(first, ts))
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in ts]
    for t, s in zip(ts, streams):
        with torch.cuda.stream(s):
            outs.append(launch(E, t))
    torch.cuda.synchronize()
    for t, out, want in zip(ts, outs, wants):
        check((out, t["k"], t["v"], None), want)
    graphs = []
    for t in ts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, launch(E, t)))
    for d, t in zip(ds, ts):
        t["k"].copy_(d["k"])
        t["v"].copy_(d["v"])
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for (_, out), t, want in zip(graphs, ts, wants):
        check((out, t["k"], t["v"], None), want)
