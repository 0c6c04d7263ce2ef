"""A decode step of rows that share a prefix (csrc/attn_shared.cu) against the formula in 64 bits.

Tolerance of a result: the final rounding to bf16, 2^-8 of it, and beside it what weights that are off by a factor 1 +- d make, 2 d sum_j w_j |v_j|, with d the sum of
  * the error of a score: hs + 2 roundings of 2^-24 of sum |q k| / sqrt(hs), in the exponent and once more in the row's maximum;
  * the rounding of the exponent's argument, 2^-23 of the largest score's distance (at most 2 max |s|), and of ex2, 2^-22;
  * a probability in two bf16 numbers: 2^-8 of it in the second one, which is rounded by 2^-8 of itself: 2^-16;
  * sums of n products in fp32: (n + 64) 2^-24, n keys at most.
The keys that the step stores are rounded as the model rounds them: bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F64 = torch.float64


@pytest.fixture(params=["list", "tensor memory", "cluster"])
def K(request):
    """The kernels with the step on one of its ways, whatever the sizes say (a cluster a group: where the group's rows are few enough)."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lit_gpt_b200 import kernels

    before = kernels.attn_decode_shared_tune({"list": 1, "tensor memory": 2, "cluster": 3}[request.param])
    yield kernels
    kernels.attn_decode_shared_tune(before)


def make(rows, groups, per, hs, prefix, cap, own, rope=None, table=torch.float32, seed=0):
    """own: tokens each row has before the step, -1 for a row that takes no part."""
    g = torch.Generator().manual_seed(seed)
    rope = hs if rope is None else rope
    angle = torch.outer(torch.arange(prefix + cap, dtype=F64), 10000.0 ** (-torch.arange(0, max(rope, 1), 2, dtype=F64)[: rope // 2] / max(rope, 1))).repeat(1, 2)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16()
    return dict(qkv=rnd(rows, (per + 2) * groups * hs), cos=angle.cos().to(table), sin=angle.sin().to(table), kc=rnd(rows, groups, cap, hs), vc=rnd(rows, groups, cap, hs),
                kp=rnd(groups, prefix, hs), vp=rnd(groups, prefix, hs), pos=torch.tensor([prefix + n if n >= 0 else -1 for n in own]), n=torch.tensor([prefix], dtype=torch.int32),
                per=per, rope=rope)


def turn(x, c, s, n):
    """apply_rope with the model's rounding points, on the CPU."""
    a = x[..., :n] if c.dtype == torch.bfloat16 else x[..., :n].float()
    other = torch.cat((-a[..., n // 2 :], a[..., : n // 2]), -1)
    return torch.cat(((a * c + other * s).bfloat16(), x[..., n:]), -1)


def formula(d, prefix_len=None):
    """-> result, bound of its error beside the final rounding, caches."""
    B, G, cap, hs = d["kc"].shape
    per, P = d["per"], d["kp"].shape[1] if prefix_len is None else prefix_len
    heads = d["qkv"].view(B, G, per + 2, hs)
    out, slack = torch.zeros(B, G, per, hs, dtype=F64), torch.zeros(B, G, per, hs, dtype=F64)
    kc, vc = d["kc"].clone(), d["vc"].clone()
    for b, p in enumerate(d["pos"].expand(B).tolist()):
        if p < 0:
            continue
        c, s = d["cos"][min(p, len(d["cos"]) - 1)], d["sin"][min(p, len(d["sin"]) - 1)]
        i = min(max(p - P, 0), cap - 1)
        kc[b, :, i], vc[b, :, i] = turn(heads[b, :, per], c, s, d["rope"]), heads[b, :, per + 1]
        q = turn(heads[b, :, :per], c, s, d["rope"]).to(F64)
        keys = torch.cat((d["kp"][:, :P], kc[b, :, : i + 1]), 1).to(F64)
        values = torch.cat((d["vp"][:, :P], vc[b, :, : i + 1]), 1).to(F64)
        score = q @ keys.transpose(1, 2) / math.sqrt(hs)
        w = torch.softmax(score, -1)
        out[b] = w @ values
        size = (q.abs() @ keys.abs().transpose(1, 2)).amax() / math.sqrt(hs)
        off = 2 * (hs + 2) * 2 ** -24 * size + 2 ** -23 * 2 * score.abs().amax() + 2 ** -22 + 2 ** -16 + (keys.shape[1] + 64) * 2 ** -24
        slack[b] = 2 * off * (w @ values.abs())
    return out.reshape(B, -1), slack.reshape(B, -1), kc, vc


def call(K, d, **kw):
    B, G, _, hs = d["kc"].shape
    t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
    t.update(kw)
    out = K.attn_decode_shared(t["qkv"], t["cos"], t["sin"], t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], G * d["per"], G, hs, d["rope"])
    return out, t["kc"], t["vc"]


def check(got, want):
    out, kc, vc = (t.cpu() for t in got)
    ref, slack, rk, rv = want
    over = (out.to(F64) - ref).abs() - (2 ** -8 * ref.abs() + slack)
    assert over.max().item() <= 0, over.max().item()
    assert torch.equal(kc, rk) and torch.equal(vc, rv)


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("rows,groups,per", [(1, 1, 1), (2, 3, 1), (5, 2, 3), (16, 2, 1), (17, 1, 2), (3, 1, 16), (2, 2, 20), (40, 1, 4), (70, 2, 4), (33, 1, 17)])
@pytest.mark.parametrize("prefix,cap", [(1, 1), (31, 7), (128, 40), (300, 130)])
def test_formula(K, hs, rows, groups, per, prefix, cap):
    own = [(5 * i + 2) % cap for i in range(rows)]
    d = make(rows, groups, per, hs, prefix, cap, own, seed=rows + prefix)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("rows,groups,per", [(10, 3, 1), (8, 2, 2), (6, 40, 3), (5, 5, 4), (4, 33, 6), (3, 148, 8), (2, 7, 14), (1, 300, 16), (1, 1, 16)])
@pytest.mark.parametrize("prefix,cap", [(0, 70), (33, 33), (700, 200)])
def test_few_rows(K, hs, rows, groups, per, prefix, cap):
    own = [-1 if i % 4 == 1 else (41 * i + cap - 1) % cap for i in range(rows)]
    d = make(rows, groups, per, hs, prefix, cap, own, seed=rows + prefix)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 127, 129, 255, 257, 511, 1000, 4097])
def test_prefix_lengths(K, prefix):
    d = make(6, 2, 4, 128, prefix, 70, [0, 1, 31, 32, 33, 69], seed=prefix)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("rows,per,hs,prefix,cap", [(64, 4, 128, 5000, 600), (100, 2, 64, 3001, 300), (2, 1, 128, 9000, 5000), (130, 1, 128, 700, 20)])
def test_long(K, rows, per, hs, prefix, cap):
    own = [(i * 37 + 1) % cap for i in range(rows - 1)] + [cap - 1]
    d = make(rows, 2, per, hs, prefix, cap, own, seed=3)
    check(call(K, d), formula(d))


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rope", [0, 2, 16, 32, 64])
def test_rotated_part(K, table, rope):
    d = make(4, 2, 2, 64, 50, 9, [0, 3, 8, -1], rope=rope, table=table, seed=rope)
    check(call(K, d), formula(d))


def test_rows_that_take_no_part(K):
    d = make(40, 2, 2, 128, 200, 30, [-1 if i % 3 else i % 30 for i in range(40)])
    check(call(K, d), formula(d))
    d["pos"] = torch.full((40,), -1)
    out, kc, vc = call(K, d)
    assert not out.any() and torch.equal(kc.cpu(), d["kc"]) and torch.equal(vc.cpu(), d["vc"])


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_one_position_for_all_and_short_prefix_on_the_device(K, kind):
    """A prefix of which only the first prefix_len positions count; what lies behind them, and behind a row's own token, may be anything."""
    d = make(5, 2, 4, 128, 64, 100, [0] * 5)
    for n, p in ((40, 41), (0, 3), (64, 64), (1, 100)):
        d["n"], d["pos"] = torch.tensor([n], dtype=kind), torch.tensor([p], dtype=kind)
        want = formula(d, n)
        e = dict(d, kp=d["kp"].clone(), vp=d["vp"].clone(), kc=d["kc"].clone(), vc=d["vc"].clone())
        e["kp"][:, n:], e["vp"][:, n:] = float("nan"), float("inf")
        e["kc"][:, :, p - n + 1 :], e["vc"][:, :, p - n + 1 :] = float("inf"), float("nan")
        out, kc, vc = call(K, e)
        check((out, torch.where(torch.arange(100)[:, None] > p - n, d["kc"], kc.cpu()), torch.where(torch.arange(100)[:, None] > p - n, d["vc"], vc.cpu())), want)


def test_positions_outside_the_caches_use_the_nearest_row(K):
    d = make(4, 1, 2, 64, 20, 8, [0] * 4)
    d["pos"] = torch.tensor([3, 19, 28, 500])
    check(call(K, d), formula(d))


def test_whole_prefix_without_a_length(K):
    d = make(3, 2, 1, 128, 77, 5, [0, 4, 2])
    check(call(K, d, n=None), formula(d))


def test_distances(K):
    """Caches and prefix that are parts of larger buffers."""
    d = make(3, 2, 4, 128, 90, 20, [0, 19, 7])
    t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
    big = torch.full((5, 3, 41, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    kc, vc = big[1:4, :2, 1:21], big.clone()[1:4, 1:, 20:40]
    kp = torch.full((4, 133, 128), float("nan"), dtype=torch.bfloat16, device="cuda")[::2, 5:95]
    vp = torch.full((2, 90, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    for view, name in ((kc, "kc"), (vc, "vc"), (kp, "kp"), (vp, "vp")):
        view.copy_(t[name])
    before = big.clone()
    got = call(K, d, kc=kc, vc=vc, kp=kp, vp=vp)
    check(got, formula(d))
    before[1:4, :2, 1:21] = kc
    assert torch.equal(big.view(torch.int16), before.view(torch.int16))   # nothing around the caches


@pytest.mark.parametrize("rows", [3, 40])
def test_infinite_values_and_keys(K, rows):
    d = make(rows, 1, 1, 128, 64, 4, [1] * rows)
    d["vp"][0, 7, 5], d["vc"][1, 0, 0, 9] = float("inf"), float("-inf")
    out = call(K, d)[0].cpu().float()
    assert (out[:, 5] == float("inf")).all() and out[1, 9] == float("-inf")
    d["kp"][0, 3] = 0
    d["vp"][0, 7, 5], d["vc"][1, 0, 0, 9] = 0, 0
    heads = d["qkv"].view(rows, 3, 128)
    d["rope"], d["cos"], d["sin"] = 0, d["cos"][:, :0], d["sin"][:, :0]
    heads[:, 0] = heads[:, 0].abs()
    d["kp"][0, 3, 0] = float("-inf")       # a key that every row scores -inf: as if it were not there
    got = call(K, d)
    d["kp"], d["vp"] = (torch.cat((t[:, :3], t[:, 4:]), 1) for t in (d["kp"], d["vp"]))
    d["n"] = torch.tensor([63])
    d["pos"] = d["pos"] - 1
    check(got, formula(d))


def test_more_rows_than_a_cta_has_threads(K):
    rows = 900
    d = make(rows, 1, 1, 64, 40, 70, [-1 if i % 7 == 3 or 300 <= i < 340 else i % 70 for i in range(rows)], seed=4)
    check(call(K, d), formula(d))


def test_offsets_past_32_bits(K):
    """The third row's cache and the third group's prefix begin behind 2^31 numbers."""
    d = make(3, 3, 2, 128, 50, 20, [7, 0, 19], seed=6)
    long = 9_000_000

    caches = []
    for t in (d["kc"], d["vc"]):
        flat = torch.empty(2 * long * 128 + 3 * 20 * 128, dtype=torch.bfloat16, device="cuda")
        view = flat.as_strided((3, 3, 20, 128), (long * 128, 20 * 128, 128, 1))
        view.copy_(t)
        caches.append(view)
    prefixes = []
    for t in (d["kp"], d["vp"]):
        flat = torch.empty(2 * long * 128 + 50 * 128, dtype=torch.bfloat16, device="cuda")
        view = flat.as_strided((3, 50, 128), (long * 128, 128, 1))
        view.copy_(t)
        prefixes.append(view)
    check(call(K, d, kc=caches[0], vc=caches[1], kp=prefixes[0], vp=prefixes[1]), formula(d))


def test_another_stream(K):
    d = make(20, 2, 4, 128, 300, 40, [i % 40 for i in range(20)], seed=9)
    t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.attn_decode_shared(t["qkv"], t["cos"], t["sin"], t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], 8, 2, 128, 128)
    side.synchronize()
    check((got, t["kc"], t["vc"]), formula(d))


def test_same_result_every_time(K):
    d = make(48, 4, 2, 128, 2100, 200, [(i * 29) % 200 for i in range(48)], seed=10)
    first = call(K, d)[0]
    for _ in range(5):
        assert torch.equal(first, call(K, d)[0])


def test_every_kernel_launch_waits_for_the_one_before(K):
    """Steps one behind the other, each on what the step before left, with and without launches that begin early."""
    for early in (True, False):
        before = K.set_pdl(early)
        try:
            d = make(6, 2, 4, 128, 200, 40, [0] * 6, seed=11)
            t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
            for i in range(12):
                t["pos"].fill_(200 + i)
                t["qkv"].copy_(d["qkv"].roll(i, 0))
                out = K.attn_decode_shared(t["qkv"], t["cos"], t["sin"], t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], 8, 2, 128, 128)
            for i in range(12):
                e = dict(d, qkv=d["qkv"].roll(i, 0), pos=torch.full((6,), 200 + i))
                want = formula(e)
                d["kc"], d["vc"] = want[2], want[3]
            check((out, t["kc"], t["vc"]), want)
        finally:
            K.set_pdl(before)


def test_scores_of_hundreds(K):
    d = make(20, 1, 2, 128, 333, 12, [i % 12 for i in range(20)])
    d["qkv"] *= 16
    check(call(K, d), formula(d))


def test_same_as_the_ordinary_step(K):
    """Prefix and own cache laid one behind the other in an ordinary cache: the ordinary step's result."""
    d = make(4, 2, 4, 128, 300, 50, [17] * 4)
    d["pos"] = torch.tensor([317])
    out, kc, vc = call(K, d)
    full = [torch.cat((a.expand(4, -1, -1, -1), b), 2).cuda() for a, b in ((d["kp"], d["kc"]), (d["vp"], d["vc"]))]
    ref = K.attn_decode(d["qkv"].cuda(), d["cos"].cuda(), d["sin"].cuda(), d["pos"].cuda(), full[0], full[1], 8, 2, 128, 128)
    ref64, slack, _, _ = formula(d)
    assert ((out.cpu().to(F64) - ref.cpu().to(F64)).abs() <= 2 * (2 ** -8 * ref64.abs() + slack)).all()
    assert torch.equal(kc, full[0][:, :, 300:]) and torch.equal(vc, full[1][:, :, 300:])


@pytest.mark.parametrize("rows", [20, 5])
def test_captured_steps_follow_position_and_length(K, rows):
    """Two graphs that are replayed on two streams at once, each with lengths that change between replays."""
    ds = [make(rows, 2, 4, 128, 600, 40, [0] * rows, seed=s) for s in (1, 2)]
    ts, graphs, outs, streams = [], [], [], [torch.cuda.Stream() for _ in ds]
    for d in ds:
        t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
        run = lambda t=t: K.attn_decode_shared(t["qkv"], t["cos"], t["sin"], t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], 8, 2, 128, 128)
        keep = t["kc"].clone(), t["vc"].clone()
        run()
        t["kc"].copy_(keep[0]), t["vc"].copy_(keep[1])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        ts.append(t), graphs.append(g), outs.append(out)
    for n, p in ((600, 600), (77, 78), (599, 638)):
        torch.cuda.synchronize()
        for d, t in zip(ds, ts):
            d["n"], d["pos"] = torch.tensor([n]), torch.full((rows,), p)
            t["n"].fill_(n), t["pos"].fill_(p)
            t["kc"].copy_(d["kc"]), t["vc"].copy_(d["vc"])
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for d, t, out in zip(ds, ts, outs):
            check((out, t["kc"], t["vc"]), formula(d, n))


def test_refusals(K):
    d = make(3, 2, 2, 64, 10, 4, [0, 1, 2])
    t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
    bad = [dict(qkv=t["qkv"][:2]), dict(qkv=t["qkv"].float()), dict(kc=t["kc"].float()), dict(kc=t["kc"].transpose(1, 2).contiguous().transpose(1, 2)), dict(vc=t["vc"][:, :, :3]),
           dict(kp=t["kp"][:1]), dict(vp=t["vp"][:, :9]), dict(kp=t["kp"].half()), dict(pos=t["pos"][:2]), dict(pos=t["pos"].float()), dict(n=torch.tensor([1, 2], device="cuda")),
           dict(n=torch.tensor([1.0], device="cuda")), dict(cos=t["cos"][:, :32]), dict(cos=t["cos"].half(), sin=t["sin"].half()), dict(kc=t["kc"][:1].expand(3, -1, -1, -1)),
           dict(pos=t["pos"].cpu()), dict(kp=torch.empty(2, 10 * 64 + 8, device="cuda", dtype=torch.bfloat16)[:, 4:-4].view(2, 10, 64))]
    for change in bad:
        with pytest.raises(K.C.B200Error):
            call(K, d, **change)
    with pytest.raises(K.C.B200Error):
        K.attn_decode_shared(t["qkv"], t["cos"], t["sin"], t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], 4, 2, 64, 64, table_preselected=True)


@pytest.mark.parametrize("rows,groups,per,prefix", [(64, 8, 4, 1700), (64, 8, 4, 1500), (20, 8, 1, 13000), (16, 8, 1, 13000), (5, 32, 1, 900), (6, 32, 1, 900), (2, 2, 4, 2000),
                                                     (2, 2, 4, 3000)])
def test_either_way_by_size(rows, groups, per, prefix):
    """Sizes on both sides of the rule: 64 x 4 rows of 8 groups over 1700 and 1500 keys, 20 and 16 rows over 13000, 5 and 6 rows, 2 x 4 rows of 2 groups
    over 2000 and 3000 keys."""
    from lit_gpt_b200 import kernels

    d = make(rows, groups, per, 128, prefix, 33, [i % 33 for i in range(rows)], seed=prefix)
    check(call(kernels, d), formula(d))


@pytest.mark.parametrize("rows,groups,per,prefix,launches", [(64, 8, 4, 1700, 4), (64, 8, 4, 1500, 3), (20, 8, 1, 13000, 4), (16, 8, 1, 13000, 3), (5, 32, 1, 900, 1), (6, 32, 1, 900, 3),
                                                              (2, 2, 4, 2000, 1), (2, 2, 4, 3000, 3)])
def test_which_way_by_size(rows, groups, per, prefix, launches):
    """The sizes of test_either_way_by_size take the way that the rule says: a cluster a group is one launch, the list three, tensor memory beside the list four."""
    from lit_gpt_b200 import kernels

    d = make(rows, groups, per, 128, prefix, 33, [i % 33 for i in range(rows)], seed=prefix)
    t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
    before = kernels.launch_count()
    kernels.attn_decode_shared(t["qkv"], t["cos"], t["sin"], t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], groups * per, groups, 128, 128)
    assert kernels.launch_count() - before == launches


@pytest.mark.parametrize("hs,rope", [(64, 64), (64, 16), (128, 128), (128, 6)])
@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_tables_by_position_in_the_call(K, hs, rope, table, rows):
    """Rows of the tables already picked, in the order of pos: one per row, rows that take no part among them, or one for all."""
    d = make(rows, 2, 2, hs, 70, 30, [-1 if i % 5 == 3 else (7 * i + 4) % 30 for i in range(rows)], rope=rope, table=table, seed=rows + rope)
    for pos in (d["pos"], torch.tensor([83])):
        d["pos"] = pos
        at = pos.clamp(min=0)
        t = {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}
        out = K.attn_decode_shared(t["qkv"], d["cos"][at].cuda(), d["sin"][at].cuda(), t["pos"], t["kc"], t["vc"], t["kp"], t["vp"], t["n"], 4, 2, hs, rope, table_preselected=True)
        check((out, t["kc"], t["vc"]), formula(d))
