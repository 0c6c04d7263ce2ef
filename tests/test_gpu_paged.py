"""Attention over a paged cache, the weights of its keys and their eviction (csrc/paged_attn.cu, csrc/paged_evict.cu) against the formulas in 64 bits (paged_oracle.py, which derives
the tolerances).  Keys that a step stores are rounded as the model rounds them: bit for bit; what an eviction leaves: bit for bit."""
import random

import pytest
import torch

import paged_oracle as oracle
from paged_oracle import F64, make

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["list", "tensor memory", "list without scores", "clusters", "by size"])
def path(request):
    return request.param


@pytest.fixture
def K(path):
    """The kernels with every sequence in the list of tiles, on the tensor memory, or where its size puts it."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lit_gpt_b200 import kernels

    before = kernels.attn_paged_tune({"list": 1, "tensor memory": 2, "list without scores": 3, "clusters": 4, "by size": 0}[path])
    yield kernels
    kernels.attn_paged_tune(before)


@pytest.fixture
def formula(path):
    """The step in 64 bits; on the tensor memory probabilities are rounded to bf16."""
    return lambda d: oracle.step(d, 0.0 if path.startswith("list") else 2 ** -8)


@pytest.fixture
def E():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lit_gpt_b200 import kernels

    return kernels


def on_gpu(d):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}


def launch(K, t, **kw):
    how = dict(max_rows=t["max_rows"], max_length=t["max_length"], key_weights=t["kw"])
    how.update(kw)
    return K.attn_paged(t["qkv"], t["cos"], t["sin"], t["row_pos"], t["row_seq"], t["seqs"], t["pages"], t["k"], t["v"], t["groups"] * t["per"], t["groups"], t["hs"], t["rope"], **how)


def call(K, d, **kw):
    t = on_gpu(d)
    out = launch(K, t, **kw)
    return out, t["k"], t["v"], t["kw"]


def same(a, b):
    """Bit for bit (NaN equal to itself)."""
    return torch.equal(a.view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32), b.view(torch.int16 if b.dtype == torch.bfloat16 else torch.int32))


def check(got, want):
    out, k, v, kw = (None if t is None else t.cpu() for t in got)
    ref, slack, rk, rv, rw, w_slack = want
    over = (out.to(F64) - ref).abs() - (2 ** -8 * ref.abs() + slack)
    assert over.max().item() <= 0, over.max().item()
    assert same(k, rk) and same(v, rv)
    if rw is not None:
        over = (kw.to(F64) - rw).abs() - w_slack
        assert over.max().item() <= 0, over.max().item()


SINGLES = [(1, 0), (1, 1), (1, 15), (1, 16), (1, 31), (1, 32), (1, 63), (1, 100), (1, 257)]
MIXED = [(1, 40), (5, 0), (0, 7), (17, 33), (1, 0), (40, 129), (2, 300)]


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("groups,per", [(1, 1), (3, 1), (2, 4), (1, 7), (2, 16), (1, 20)])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("steps", [SINGLES, MIXED, [(70, 0)], [(33, 90), (64, 0)]], ids=["singles", "mixed", "prompt", "chunks"])
def test_formula(K, formula, hs, groups, per, page, steps):
    d = make(steps, groups, per, hs, page, seed=page + per)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("per,hs", [(70, 64), (130, 128)])
def test_many_heads_a_group(K, formula, per, hs):
    d = make([(1, 50), (3, 0), (1, 200)], 1, per, hs, 32, seed=per)
    check(call(K, d), formula(d))


def test_registered_operator(K, formula):
    from lit_gpt_b200 import ops  # noqa: F401

    d = make([(1, 50), (30, 7)], 2, 2, 64, 16)
    t = on_gpu(d)
    out = torch.ops.b200gpt.attn_paged(t["qkv"], t["cos"], t["sin"], t["row_pos"], t["row_seq"], t["seqs"], t["pages"], t["k"], t["v"], 4, 2, 64, 64, t["max_rows"], t["max_length"], t["kw"])
    check((out, t["k"], t["v"], t["kw"]), formula(d))


@pytest.mark.parametrize("hs,groups,per", [(64, 1, 1), (128, 3, 4), (64, 2, 8), (128, 2, 9), (64, 1, 16), (128, 2, 1)])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("cached", [[0], [1, 31, 32], [500], [900, 0, 63, 1300, 64], [127] * 9])
def test_single_tokens_without_weights(K, formula, hs, groups, per, page, cached):
    d = make([(1, n) for n in cached], groups, per, hs, page, weights=False, seed=len(cached))
    check(call(K, d), formula(d))
    d["seqs"][0, 1] = 0                         # a sequence without a row, a row without a sequence
    d["row_seq"][0] = -1
    check(call(K, d), formula(d))
    if len(cached) > 1:
        d["pages"][d["seqs"][1, 3], 0] = -1     # a missing page
        d["pages"][d["seqs"][-1, 3], (cached[-1]) // page] = 2 ** 30   # the new key's
        check(call(K, d), formula(d))


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 200, 257])
def test_chunk_lengths(K, formula, rows):
    d = make([(rows, rows * 3 % 50)], 2, 4, 128, 64, seed=rows)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("steps", [[(1, 5000)], [(1, 3), (1, 4097), (1, 900)], [(1, 17 * i) for i in range(70)], [(130, 1500)]])
@pytest.mark.parametrize("per,hs", [(4, 128), (1, 64)])
def test_long(K, formula, steps, per, hs):
    d = make(steps, 2, per, hs, 64, seed=3)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("rows,cached,per,hs", [(3000, 4100, 3, 64), (1300, 2000, 8, 128), (4000, 0, 1, 128)])
def test_weights_of_long_chunks(E, rows, cached, per, hs):
    """Many tiles of queries for every key.  The formula on the GPU in 64 bits, from the keys that the step has stored; the bound as in paged_oracle."""
    G, page = 2, 64
    d = make([(rows, cached)], G, per, hs, page, seed=rows)
    t = on_gpu(d)
    before = t["kw"].clone()
    out = launch(E, t)
    at = t["pages"][d["seqs"][0, 3]].long()
    n = rows + cached
    ids, slots = at[torch.arange(n, device="cuda") // page], torch.arange(n, device="cuda") % page
    keys = t["k"][ids, :, slots].to(F64)                                   # (n, G, hs)
    heads = t["qkv"].view(rows, G, per + 2, hs)
    q = oracle.turn(heads[:, :, :per], t["cos"][cached:][:, None, None], t["sin"][cached:][:, None, None], hs).to(F64)
    got, err = torch.zeros(n, G, dtype=F64, device="cuda"), torch.zeros(n, G, dtype=F64, device="cuda")
    for lo in range(0, rows, 250):
        hi = min(lo + 250, rows)
        s = torch.einsum("igph,jgh->gpij", q[lo:hi], keys) / hs ** 0.5
        size = torch.einsum("igph,jgh->gpij", q[lo:hi].abs(), keys.abs()).amax() / hs ** 0.5
        s = s.masked_fill(torch.arange(n, device="cuda") > cached + torch.arange(lo, hi, device="cuda")[:, None], float("-inf"))
        w = torch.softmax(s, -1).sum((1, 2)).T
        off = 2 * (hs + 2) * 2 ** -24 * size + 2 ** -23 * 2 * s[s > float("-inf")].abs().amax() + 2 ** -22 + (n + 64) * 2 ** -24
        got += w
        err += 2 * off * w
    old = before[ids, :, slots].to(F64)
    old[cached:] = 0
    over = (t["kw"][ids, :, slots].to(F64) - (old + got)).abs() - err - (rows * per + 8) * 2 ** -24 * (old + got)
    assert over.max().item() <= 0, over.max().item()
    again = on_gpu(d)
    assert same(out, launch(E, again)) and same(t["kw"], again["kw"])


def test_many_sequences(K, formula):
    """More sequences than a CTA has threads."""
    d = make([(1 if i % 3 else 0, i % 50) for i in range(1500)], 1, 2, 64, 16, seed=4)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("n", [31, 32, 33, 319, 321, 513])
def test_as_many_sequences_as_a_list_is_cut_by(K, formula, n):
    """A warp's number of sequences, a CTA's, one more: chunks and tokens, some without rows, the longest last."""
    d = make([(0 if i % 5 == 2 else 1 + i % 4 * 3, i * 7 % 40) for i in range(n - 1)] + [(70, 90)], 2, 4, 64, 16, seed=n)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rope", [0, 2, 16, 32, 64])
def test_rotated_part(K, formula, table, rope):
    d = make([(1, 9), (20, 13)], 2, 2, 64, 16, rope=rope, table=table, seed=rope)
    check(call(K, d), formula(d))


def test_without_weights(K, formula):
    d = make(MIXED, 2, 2, 128, 32, weights=False)
    check(call(K, d), formula(d))


def test_positions_apart_from_places(K, formula):
    """A cache that was cut down: rows are rotated at their positions, which are not their places in the cache; positions in 64 bits; tables gathered before the call."""
    d = make([(1, 9), (20, 13)], 2, 2, 64, 16, seed=9)
    d["cos"], d["sin"] = (torch.cat([t] * 9) for t in (d["cos"], d["sin"]))
    d["row_pos"] = (d["row_pos"].long() * 7 + 3) % len(d["cos"])
    want = formula(d)
    check(call(K, d), want)
    d["cos"], d["sin"] = d["cos"][d["row_pos"]], d["sin"][d["row_pos"]]
    check(call(K, d, table_preselected=True), want)


def test_leading_dimensions_and_strided_rows(K, formula):
    d = make([(1, 9), (21, 13)], 2, 2, 64, 16, seed=9)
    want = formula(d)
    t = on_gpu(d)
    wide = torch.zeros(2, 11, 600, device="cuda", dtype=torch.bfloat16)
    wide[..., :512] = t["qkv"].view(2, 11, 512)
    t["qkv"] = wide[..., :512]
    apart = torch.full((len(d["pages"]), 30), 77, device="cuda", dtype=torch.int32)   # a wider page table
    apart[:, : d["pages"].shape[1]] = t["pages"]
    t["pages"] = apart[:, : d["pages"].shape[1]]
    out = launch(K, t)
    assert out.shape == (22, 4 * 64)
    check((out, t["k"], t["v"], t["kw"]), want)


@pytest.mark.parametrize("layout", ["keys beside values", "group by group", "apart"])
def test_page_layouts(K, formula, layout):
    d = make(MIXED, 3, 2, 128, 32, seed=12)
    want = formula(d)
    t = on_gpu(d)
    P, G, page, hs = d["k"].shape
    if layout == "keys beside values":
        both = torch.empty(P, 2, G, page, hs, device="cuda", dtype=torch.bfloat16)
        k, v = both[:, 0], both[:, 1]
    elif layout == "group by group":
        k, v = (torch.empty(G, P, page, hs, device="cuda", dtype=torch.bfloat16).transpose(0, 1) for _ in range(2))
    else:
        k, v = (torch.empty(P * (G * page * hs + 64) + 64, device="cuda", dtype=torch.bfloat16).as_strided((P, G, page, hs), (G * page * hs + 64, page * hs + 8, hs, 1)) for _ in range(2))
        k, v = (x.as_strided((P, G, page, hs), (G * page * hs + 64, page * hs + 8, hs, 1)) for x in (k, v))
    k.copy_(t["k"])
    v.copy_(t["v"])
    t["k"], t["v"] = k, v
    out = launch(K, t)
    check((out, k.contiguous(), v.contiguous(), t["kw"]), want)


def test_missing_pages(K, formula):
    """No page: no keys there, new ones are dropped; a row without any key has a result of zero.  Page numbers outside the pool are none."""
    d = make([(1, 100), (1, 100), (30, 50), (3, 20), (1, 16)], 2, 4, 128, 16, seed=5)
    at = d["seqs"][:, 3].tolist()
    d["pages"][at[0], 2] = -1
    d["pages"][at[1], 6] = len(d["k"])          # the new key's
    d["pages"][at[2], 3] = -7                   # within the chunk
    d["pages"][at[2], 0] = 2 ** 31 - 1
    d["pages"][at[3]] = -1                      # all of them
    d["pages"][at[4], 0] = -1
    want = formula(d)
    got = call(K, d)
    check(got, want)
    assert not got[0][32:35].any()


def test_bounds_drop_keys(K, formula):
    """Keys from max_length on are dropped; the rows behind see those before."""
    d = make([(1, 60), (20, 50)], 2, 2, 64, 16, seed=6)
    d["max_length"] = 60
    check(call(K, d), formula(d))


def test_rows_of_no_sequence(K, formula):
    d = make([(1, 20), (6, 10), (1, 5)], 2, 2, 64, 16, seed=7)
    want = [t.clone() if torch.is_tensor(t) else t for t in formula({**d, "seqs": torch.cat((d["seqs"][:2], d["seqs"][2:] * torch.tensor([1, 0, 1, 1], dtype=torch.int32)))})]
    d["row_seq"][7] = -1
    bad = d["seqs"].clone()
    bad[2] = torch.tensor([0, 0, 5, 0])
    d["seqs"] = bad.int()
    got = call(K, d)
    check(got, want)
    assert not got[0][7].any()


@pytest.mark.parametrize("seq", [(0, 500, 3, 0), (-1, 2, 3, 0), (7, 1, -2, 0), (7, 1, 3, 99), (7, 1, 3, -1), (2 ** 31 - 1, 2 ** 31 - 1, 5, 0), (7, 1, 2 ** 31 - 1, 0)])
def test_sequences_that_do_not_fit_take_no_part(K, formula, seq):
    """A description that reaches beyond the rows or the page table: nothing of it is read or written."""
    d = make([(1, 20), (6, 10), (1, 5)], 2, 2, 64, 16, seed=7)
    want = formula({**d, "seqs": torch.cat((d["seqs"][:2], torch.zeros(1, 4, dtype=torch.int32)))})
    d["seqs"][2] = torch.tensor(seq, dtype=torch.int32)
    got = call(K, d)
    if seq[2] < 2 ** 31 - 1:
        check(got, want)
    else:                                       # as many cached keys as there is no room for: the row sees all the places, of which it has no pages but its own
        assert torch.isfinite(got[0].float()).all() and same(got[1].cpu(), want[2])


def test_what_lies_behind_the_last_key_is_not_read(K, formula):
    for steps in (SINGLES, [(20, 33), (1, 70)]):
        d = make(steps, 2, 4, 128, 64, seed=8)
        want = formula(d)
        used = torch.zeros(d["k"].shape[0], d["k"].shape[2], dtype=torch.bool)
        for first, rows, cached, at in d["seqs"].tolist():
            for j in range(cached + rows):
                used[d["pages"][at, j // 64], j % 64] = True
        for x, bad in ((d["k"], float("nan")), (d["v"], float("inf"))):
            x.permute(0, 2, 1, 3)[~used] = bad
        want = (want[0], want[1], *formula(d)[2:4], want[4], want[5])
        check(call(K, d), want)


def test_offsets_past_32_bits(K, formula):
    """Pages more than 2^31 numbers into the pool."""
    d = make([(1, 40), (20, 70)], 1, 2, 128, 256, seed=10)
    want = formula(d)
    t = on_gpu(d)
    P, far = len(d["k"]), 2 ** 31 // (256 * 128) + 5
    k, v = (torch.empty(far + P, 1, 256, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kw = torch.zeros(far + P, 1, 256, device="cuda")
    k[far:], v[far:], kw[far:] = t["k"], t["v"], t["kw"]
    t.update(k=k, v=v, kw=kw, pages=torch.where(t["pages"] >= 0, t["pages"] + far, -1).int())
    out = launch(K, t)
    check((out, k[far:], v[far:], kw[far:]), want)


def test_same_bits_every_time(K, formula):
    d = make([(1, 700), (64, 300), (1, 90), (200, 0)], 2, 4, 128, 64, seed=11)
    first = call(K, d)
    for _ in range(3):
        for a, b in zip(first, call(K, d)):
            assert same(a, b)


def test_two_streams(K, formula):
    """Two calls at a time share nothing."""
    ds = [make([(1, 300 + 50 * i), (1 + 30 * i, 20)], 2, 4, 128, 32, seed=20 + i) for i in range(2)]
    wants = [formula(d) for d in ds]
    ts = [on_gpu(d) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    outs = []
    for _ in range(1):
        for t, s in zip(ts, streams):
            with torch.cuda.stream(s):
                outs.append(launch(K, t))
    torch.cuda.synchronize()
    for t, out, want in zip(ts, outs, wants):
        check((out, t["k"], t["v"], t["kw"]), want)


def test_captured_steps(K, formula):
    """A captured step follows its description, page table and positions as they change; two captured steps at a time have a workspace each."""
    first = make([(1, 40), (1, 100), (1, 9)], 2, 4, 128, 16, seed=30)
    second = make([(1, 250), (0, 3), (1, 77)], 2, 4, 128, 16, seed=31, spare=2)
    longest = 300
    for d in (first, second):
        d["max_length"] = longest
        d["pages"] = torch.nn.functional.pad(d["pages"], (0, 20 - d["pages"].shape[1]), value=-1)
        pad = 30 - len(d["k"])
        for name in ("k", "v", "kw"):
            d[name] = torch.cat((d[name], d[name][:1].repeat(pad, *[1] * (d[name].dim() - 1))))
    second["qkv"] = torch.cat((second["qkv"][:1], second["qkv"][:1], second["qkv"][1:]))
    second["row_seq"] = torch.tensor([0, -1, 2], dtype=torch.int32)
    second["row_pos"] = torch.tensor([250, 0, 77], dtype=torch.int32)
    second["seqs"] = torch.tensor([[0, 1, 250, second["seqs"][0, 3]], [1, 0, 3, second["seqs"][1, 3]], [2, 1, 77, second["seqs"][2, 3]]], dtype=torch.int32)
    first["cos"], first["sin"] = second["cos"], second["sin"]
    want = [formula(d) for d in (first, second)]
    t = on_gpu(first)
    launch(K, t)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = launch(K, t)
        graphs.append((g, out))
    for d, w in zip((first, second), want):
        for name in ("qkv", "row_pos", "row_seq", "seqs", "pages"):
            t[name].copy_(d[name])
        for g, out in graphs:
            for name in ("k", "v", "kw"):
                t[name].copy_(d[name])
            g.replay()
            torch.cuda.synchronize()
            check((out, t["k"], t["v"], t["kw"]), w)


# ---- eviction ----------------------------------------------------------------------------------------------------------------------
def cache(lengths, groups, hs, page, seed=0, spare=2):
    d = make([(0, n) for n in lengths], groups, 1, hs, page, seed=seed, spare=spare)
    return d, [int(at) for at in d["seqs"][:, 3]]


def evict_check(E, d, lengths, keep, rows, **kw):
    want = oracle.evict(d["k"], d["v"], d["kw"], d["pages"], lengths, keep, rows=rows, **kw)
    t = on_gpu(d)
    left = E.evict_paged(t["k"], t["v"], t["kw"], t["pages"], torch.tensor(lengths, dtype=torch.int32, device="cuda"), keep, max_length=max(max(lengths), 1),
                         rows=None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda"), **kw)
    assert same(t["k"].cpu(), want[0]) and same(t["v"].cpu(), want[1]) and same(t["kw"].cpu(), want[2]) and left.tolist() == want[3]


@pytest.mark.parametrize("hs,groups,page", [(64, 1, 16), (128, 3, 64), (64, 2, 256), (128, 2, 32)])
@pytest.mark.parametrize("lengths,keep,first,recent", [([2], 1, 0, 0), ([100], 99, 0, 0), ([100], 1, 1, 0), ([100, 7, 300], 50, 4, 16), ([1025, 2, 1024, 1023], 64, 0, 64),
                                                       ([1500], 1400, 64, 300), ([513, 40, 41], 40, 0, 7), ([2100, 2049], 700, 1, 0), ([33], 32, 16, 16)])
def test_evict(E, hs, groups, page, lengths, keep, first, recent):
    d, rows = cache(lengths, groups, hs, page, seed=keep)
    evict_check(E, d, lengths, keep, rows, first=first, recent=recent)


@pytest.mark.parametrize("lengths,keep,first,recent", [([9000, 5000], 4097, 5, 1000), ([60000, 500, 41000], 33333, 5, 100), ([60000], 100, 0, 0)])
def test_evict_long(E, lengths, keep, first, recent):
    """Weights that fit into shared memory and such that do not."""
    d, rows = cache(lengths, 1, 64, 16, seed=3)
    d["kw"] = (d["kw"] * 1000).round() / 1000          # (equal ones among them)
    evict_check(E, d, lengths, keep, rows, first=first, recent=recent)


@pytest.mark.parametrize("hs,groups,page,lengths,keep,first,recent",
                         [(64, 1, 16, [16385], 16384, 0, 0), (128, 1, 16, [17001, 2, 17], 1, 0, 0), (64, 2, 16, [20003], 77, 70, 7), (128, 2, 256, [16411, 2100, 1999], 1999, 1500, 400),
                          (64, 1, 32, [18191, 300], 299, 0, 299), (128, 1, 64, [7, 17777, 9], 6, 2, 1), (64, 18, 64, [17000, 30], 1000, 1, 30), (64, 19, 64, [17000, 30], 1000, 1, 30),
                          (64, 38, 64, [17000, 30], 1000, 1, 30)])
def test_evict_chosen_together(E, hs, groups, page, lengths, keep, first, recent):
    """Few sequences of more keys than a thread block chooses from by itself; some of them are so short that parts of the cluster have none of their keys."""
    d, rows = cache(lengths, groups, hs, page, seed=keep)
    d["kw"] = (d["kw"] * 100).round() / 100            # (equal ones among them, on both sides of a part's end)
    evict_check(E, d, lengths, keep, rows, first=first, recent=recent)


@pytest.mark.parametrize("kind", ["zeros", "few values", "not a number", "neighbours"])
def test_evict_chosen_together_ties(E, kind):
    lengths = [17300, 900]
    d, rows = cache(lengths, 1, 64, 32, seed=23)
    r = torch.Generator().manual_seed(2)
    pick = lambda *values: torch.tensor(values)[torch.randint(len(values), d["kw"].shape, generator=r)]
    nan, inf = float("nan"), float("inf")
    d["kw"] = {"zeros": lambda: torch.zeros_like(d["kw"]), "few values": lambda: pick(0.0, 1.0, 2.5), "not a number": lambda: pick(nan, inf, 1.0, -nan, -2.0),
               "neighbours": lambda: 1.0 + torch.randint(0, 600, d["kw"].shape, generator=r) * 2 ** -23}[kind]().float()
    for keep in (17299, 899, 40):
        evict_check(E, d, lengths, keep, rows, first=3, recent=20)


def test_evict_chosen_together_leaves_what_it_must(E):
    """An entry that is no page, a length of more than max_length, a row outside the table: in clusters too the sequence stays."""
    lengths = [2200, 2100, 20400]
    d, rows = cache(lengths, 2, 64, 64, seed=25)
    d["pages"][rows[1], 30] = len(d["k"])
    want = oracle.evict(d["k"], d["v"], d["kw"], d["pages"], lengths[:2], 600, rows=rows[:2])
    t = on_gpu(d)
    left = E.evict_paged(t["k"], t["v"], t["kw"], t["pages"], torch.tensor(lengths + [2200, 0, -5], dtype=torch.int32, device="cuda"), 600, max_length=20000,
                         rows=torch.tensor(rows + [-1, rows[0], rows[0]], dtype=torch.int32, device="cuda"))
    assert left.tolist() == [600, 2100, 20400, 2200, 0, -5]
    assert same(t["k"].cpu(), want[0]) and same(t["v"].cpu(), want[1]) and same(t["kw"].cpu(), want[2])


@pytest.mark.parametrize("lengths,groups,keep,max_length", [([2100, 40, 900, 1500] + [33] * 34, 2, 700, 60000), ([60000], 1, 49000, 60000)])
def test_evict_in_two_launches(E, lengths, groups, keep, max_length):
    """Weights that fit into no thread block's shared memory, nor into a cluster's beside the places."""
    d, rows = cache(lengths, groups, 64, 16, seed=29)
    d["kw"] = (d["kw"] * 100).round() / 100
    d["pages"] = torch.nn.functional.pad(d["pages"], (0, max(0, max_length // 16 - d["pages"].shape[1])), value=-1)
    want = oracle.evict(d["k"], d["v"], d["kw"], d["pages"], lengths, keep, rows=rows, first=5, recent=50)
    t = on_gpu(d)
    left = E.evict_paged(t["k"], t["v"], t["kw"], t["pages"], torch.tensor(lengths, dtype=torch.int32, device="cuda"), keep, max_length=max_length, first=5, recent=50,
                         rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
    assert same(t["k"].cpu(), want[0]) and same(t["v"].cpu(), want[1]) and same(t["kw"].cpu(), want[2]) and left.tolist() == want[3]


@pytest.mark.parametrize("kind", ["zeros", "few values", "signs", "infinite", "not a number", "neighbours", "tiny"])
def test_evict_ties_and_odd_weights(E, kind):
    """Equal weights: the lower index; the two zeros are equal; NaN above all."""
    lengths = [700, 300]
    d, rows = cache(lengths, 2, 64, 32, seed=17)
    r = torch.Generator().manual_seed(1)
    pick = lambda *values: torch.tensor(values)[torch.randint(len(values), d["kw"].shape, generator=r)]
    nan, inf = float("nan"), float("inf")
    d["kw"] = {"zeros": lambda: torch.zeros_like(d["kw"]), "few values": lambda: pick(0.0, 1.0, 2.5), "signs": lambda: pick(0.0, -0.0, -1.0, 1e-30, -1e-30),
               "infinite": lambda: pick(inf, -inf, 0.0, 3.0), "not a number": lambda: pick(nan, inf, 1.0, -nan, -2.0),
               "neighbours": lambda: 1.0 + torch.randint(0, 600, d["kw"].shape, generator=r) * 2 ** -23, "tiny": lambda: torch.randint(0, 300, d["kw"].shape, generator=r) * 2.0 ** -149}[kind]().float()
    for keep in (299, 128, 57):
        evict_check(E, d, lengths, keep, rows, first=3, recent=20)


def test_evict_leaves_what_it_must(E):
    """Sequences that are short, longer than max_length, or with an entry that is no page, stay as they are; as do those that are in no row of the page table."""
    lengths = [300, 40, 300, 500, 90]
    d, rows = cache(lengths, 2, 64, 16, seed=18)
    d["pages"][rows[2], 18] = -1
    want = oracle.evict(d["k"], d["v"], d["kw"], d["pages"], lengths, 64, rows=rows)
    k, v, kw, _ = oracle.evict(d["k"], d["v"], d["kw"], d["pages"], lengths[:3] + lengths[4:], 64, rows=rows[:3] + rows[4:])
    t = on_gpu(d)
    left = E.evict_paged(t["k"], t["v"], t["kw"], t["pages"], torch.tensor(lengths + [300], dtype=torch.int32, device="cuda"), 64, max_length=400,
                         rows=torch.tensor(rows + [77], dtype=torch.int32, device="cuda"))
    assert left.tolist() == [64, 40, 300, 500, 64, 300] and want[3] == [64, 40, 300, 64, 64]
    assert same(t["k"].cpu(), k) and same(t["v"].cpu(), v) and same(t["kw"].cpu(), kw)
    before = [x.clone() for x in (t["k"], t["v"], t["kw"])]
    left = E.evict_paged(t["k"], t["v"], t["kw"], t["pages"], torch.tensor(lengths, dtype=torch.int32, device="cuda"), 512, max_length=500)
    assert left.tolist() == lengths and all(same(a, b) for a, b in zip(before, (t["k"], t["v"], t["kw"])))


def test_evict_captured_and_on_another_stream(E):
    lengths = [200, 150]
    d, rows = cache(lengths, 2, 64, 16, seed=19)
    want = oracle.evict(d["k"], d["v"], d["kw"], d["pages"], lengths, 100, first=2, recent=9, rows=rows)
    t = on_gpu(d)
    n, r = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, rows))
    run = lambda: E.evict_paged(t["k"], t["v"], t["kw"], t["pages"], n, 100, first=2, recent=9, max_length=200, rows=r)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        left = run()
    torch.cuda.synchronize()
    assert same(t["k"].cpu(), want[0]) and left.tolist() == want[3]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        left = run()
    for name in ("k", "v", "kw"):
        t[name].copy_(d[name])
    g.replay()
    assert same(t["k"].cpu(), want[0]) and same(t["v"].cpu(), want[1]) and same(t["kw"].cpu(), want[2]) and left.tolist() == want[3]


# ---- the operators together ------------------------------------------------------------------------------------------------------------
def test_a_sequence_of_steps(K, formula):
    """A prompt in portions, tokens one by one, an eviction, more tokens: as a server uses them.  The choice of an eviction is made from the kernels' own weights."""
    G, per, hs, page = 2, 4, 64, 16
    r = random.Random(3)
    lengths, positions = [0, 0, 0], [0, 0, 0]
    pages = torch.full((3, 12), -1, dtype=torch.int32)
    order = list(range(36))
    r.shuffle(order)
    for i in range(3):
        pages[i] = torch.tensor(order[12 * i : 12 * i + 12])
    base = make([(1, 400)], G, per, hs, page)
    pool = dict(k=torch.zeros(36, G, page, hs).bfloat16(), v=torch.zeros(36, G, page, hs).bfloat16(), kw=torch.zeros(36, G, page))
    gpu = on_gpu(pool)
    g = torch.Generator().manual_seed(8)
    for n, step in enumerate([[50, 3, 70], [30, 1, 20], [1, 1, 1], [1, 60, 0], [1, 1, 1], "evict", [1, 1, 1], [40, 0, 1], "evict", [1, 1, 1]]):
        if step == "evict":
            want = oracle.evict(pool["k"], pool["v"], gpu["kw"].cpu(), pages, lengths, 40, first=2, recent=8)
            left = K.evict_paged(gpu["k"], gpu["v"], gpu["kw"], pages.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), 40, first=2, recent=8, max_length=192)
            pool["k"], pool["v"], pool["kw"], lengths = want
            assert left.tolist() == lengths and same(gpu["k"].cpu(), pool["k"]) and same(gpu["v"].cpu(), pool["v"]) and same(gpu["kw"].cpu(), pool["kw"])
            continue
        seqs, row_seq, row_pos = [], [], []
        for i, rows in enumerate(step):
            seqs.append((len(row_seq), rows, lengths[i], i))
            row_seq += [i] * rows
            row_pos += range(positions[i], positions[i] + rows)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)
        d = dict(base, **pool, qkv=torch.randn(len(row_seq), (per + 2) * G * hs, generator=g).bfloat16(), row_seq=i32(row_seq), row_pos=i32(row_pos), seqs=i32(seqs), pages=pages,
                 max_rows=max(step), max_length=192)
        want = formula(d)
        t = dict(on_gpu(d), **gpu)
        out = launch(K, t)
        check((out, gpu["k"], gpu["v"], gpu["kw"]), want)
        pool = dict(k=want[2], v=want[3], kw=gpu["kw"].cpu())     # (the weights: the kernels' own from here on)
        lengths = [a + b for a, b in zip(lengths, step)]
        positions = [a + b for a, b in zip(positions, step)]
