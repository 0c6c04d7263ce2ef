"""Penalties, biases and masks on logits and the draw of a token per row (csrc/logits.cu).

The adjusted logits are fp32 numbers with every step rounded by itself: numpy's fp32 gives them bit for bit.  The draw is compared with the formula in 64 bits on those
numbers: tokens are equal.  Tolerance of a log-probability: a term of the sum is off by 2^-22 (exp2), 2^-23 of its exponent (where it is small it counts as little), the
sum's additions by 2^-24 each over a thread's at most 128 terms and a warp's 5: 2^-22 (1 + 24) + 140 * 2^-24 < 2^-16 of the sum, hence of its logarithm absolutely, and the final
rounding 2^-24 of the value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lit_gpt_b200 import kernels

    return kernels


def make(B, V, dtype=torch.float32, seed=0, counts=True, bias="rows", allowed="rows", scale=3.0):
    g = torch.Generator().manual_seed(seed)
    d = dict(logits=(torch.randn(B, V, generator=g) * scale).to(dtype))
    if counts:
        d["counts"] = (torch.rand(B, V, generator=g) < 0.2).int() * torch.randint(-2, 30, (B, V), generator=g, dtype=torch.int32)
    if bias:
        d["bias"] = torch.randn(*((V,) if bias == "one" else (B, V)), generator=g)
    if allowed:
        d["ok"] = torch.rand(*((V,) if allowed == "one" else (B, V)), generator=g) < 0.5
        d["ok"][..., V // 2] = True
    d.update(repetition=1.0 + torch.rand(B, generator=g), frequency=torch.rand(B, generator=g), presence=torch.rand(B, generator=g))
    return d


def adjusted(d):
    l = d["logits"].float().numpy()
    with np.errstate(all="ignore"):
        if "counts" in d:
            n = d["counts"].numpy()
            rep, freq, pres = (np.float32(d[k].numpy()[:, None]) if torch.is_tensor(d[k]) else np.float32(d[k]) for k in ("repetition", "frequency", "presence"))
            less = np.where(l > 0, l / rep, l * rep) - freq * n.astype(np.float32)
            l = np.where(n > 0, less - pres, l)
        if "bias" in d:
            l = l + d["bias"].numpy()
        if "ok" in d:
            l = np.where(d["ok"].numpy(), l, np.float32(-np.inf))
    return l


def rules(K, d):
    kw = {k: d[k].cuda() if torch.is_tensor(d[k]) else d[k] for k in ("counts", "bias", "repetition", "frequency", "presence") if k in d}
    if "ok" in d:
        kw["allowed"] = K.pack_allowed(d["ok"].cuda())
    return kw


def drawn(l, T, k, e):
    """Token and log-probability of one row in 64 bits."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    if l.max() == -np.inf:
        return -1, -np.inf
    greedy = not T > 0
    order = np.argsort(-l, kind="stable")[: len(l) if greedy or k <= 0 else k]
    order = order[l[order] > -np.inf]
    with np.errstate(all="ignore"):
        w = np.where(l[order] == l[order[0]], 0.0, (l[order] - l[order[0]]) / (1.0 if greedy else float(T)))
        score = w if greedy else w - np.log(e[order].astype(np.float64))
    at = np.flatnonzero(score == score.max())
    at = at[np.argmin(order[at])]
    return int(order[at]), w[at] - np.log(np.exp(w).sum())


def check_draw(K, d, T, k, e, logits=None, **more):
    l = adjusted(d)
    B = len(l)
    tok, lp = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, device="cuda")
    on = lambda x: x.cuda() if torch.is_tensor(x) else x
    K.sample_rows_(d["logits"].cuda() if logits is None else logits, tok, on(T), on(k), noise=on(e), logprob_out=lp, **rules(K, d), **more)
    for b in range(B):
        want = drawn(l[b], T[b].item() if torch.is_tensor(T) else T, k[b].item() if torch.is_tensor(k) else k or 0, None if e is None else e.expand(B, -1)[b].numpy())
        assert tok[b].item() == want[0], (b, tok[b].item(), want)
        if want[0] >= 0:
            assert abs(lp[b].item() - want[1]) <= 2 ** -16 + 2 ** -24 * abs(want[1]), (b, lp[b].item(), want)
        else:
            assert lp[b].item() == -float("inf")
    return tok, lp


def exponential(*shape, seed=1):
    return torch.empty(*shape).exponential_(1, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 31), (2, 33), (5, 1000), (4, 4099), (7, 50257), (2, 32000), (64, 130)])
@pytest.mark.parametrize("bias,allowed", [("", ""), ("one", "rows"), ("rows", "one")])
def test_adjusted(K, dtype, B, V, bias, allowed):
    d = make(B, V, dtype, seed=V, bias=bias, allowed=allowed)
    want = torch.from_numpy(np.ascontiguousarray(adjusted(d)))
    got = K.adjust_logits(d["logits"].cuda(), **rules(K, d))
    assert got.dtype == torch.float32 and torch.equal(got.cpu(), want)
    there = d["logits"].cuda()
    assert K.adjust_logits(there, **rules(K, d), out=there) is there and torch.equal(there.cpu(), want.to(dtype))
    wide = torch.full((B, V + 3), 7.0, device="cuda", dtype=torch.bfloat16)
    K.adjust_logits(d["logits"].cuda(), **rules(K, d), out=wide[:, 1 : V + 1])
    assert torch.equal(wide[:, 1 : V + 1].cpu(), want.bfloat16()) and (wide[:, 0] == 7).all() and (wide[:, V + 1 :] == 7).all()


def test_adjusted_numbers_for_all_rows_and_none(K):
    d = make(3, 500)
    d.update(repetition=1.3, frequency=0.25, presence=-0.5)
    assert torch.equal(K.adjust_logits(d["logits"].cuda(), **rules(K, d)).cpu(), torch.from_numpy(np.ascontiguousarray(adjusted(d))))
    assert torch.equal(K.adjust_logits(d["logits"].cuda()).cpu(), d["logits"])


def test_adjusted_infinities_and_nan(K):
    d = make(2, 64, allowed="")
    d["logits"][0, :6] = torch.tensor([float("inf"), float("-inf"), float("nan"), float("inf"), float("-inf"), float("nan")])
    d["counts"][0, :3], d["counts"][0, 3:6] = 2, 0
    d["bias"][1, 5], d["bias"][1, 6] = float("-inf"), float("inf")
    want = torch.from_numpy(np.ascontiguousarray(adjusted(d)))
    assert torch.equal(K.adjust_logits(d["logits"].cuda(), **rules(K, d)).cpu().nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))
    d["ok"] = torch.zeros(2, 64, dtype=torch.bool)
    assert (K.adjust_logits(d["logits"].cuda(), **rules(K, d)) == -float("inf")).all()


def test_rows_at_a_distance_and_one_row_for_all(K):
    d = make(4, 1001)
    big = torch.full((4, 1024), float("nan"), device="cuda")
    big[:, 3:1004] = d["logits"].cuda()
    e = exponential(4, 1001)
    T = torch.tensor([0.7, 0.0, 1.1, 2.0])
    check_draw(K, d, T, 50, e, logits=big[:, 3:1004])
    d["logits"] = d["logits"][:1].expand(4, -1)
    one = d["logits"][:1].cuda().expand(4, -1)
    assert torch.equal(K.adjust_logits(one, **rules(K, d)).cpu(), torch.from_numpy(np.ascontiguousarray(adjusted(d))))
    check_draw(K, d, T, 50, e, logits=one)
    d["logits"] = torch.randn(1001, 4).T
    check_draw(K, d, T, 50, e, logits=d["logits"].cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 1), (2, 3), (3, 37), (4, 2049), (1, 32000), (5, 50257), (150, 4100), (300, 600)])
@pytest.mark.parametrize("k", [None, 1, 2, 40, 200])
def test_draw(K, dtype, B, V, k):
    d = make(B, V, dtype, seed=B + V + (k or 0), counts=k != 40, bias="" if k == 1 else "one", allowed="rows" if k == 200 else "")
    T = 0.5 + torch.rand(B, generator=torch.Generator().manual_seed(7))
    T[B // 2] = 0.0
    check_draw(K, d, T, k, exponential(B, V, seed=V))


def test_draw_large_vocabularies(K):
    for V in (200001, 500001):    # slices that do and do not fit shared memory
        d = make(2, V, counts=False, bias="", allowed="rows")
        for k in (0, 3, 5000):
            check_draw(K, d, 0.9, k, exponential(2, V, seed=k))
        check_draw(K, d, 0.0, 0, None)


def test_log_probabilities_of_near_certain_tokens(K):
    """One logit far above the others: ln p = -ln(1 + d), d the others' weights, of which each is off by 2^-22 (ex2), its exponent's rounding being carried along, and the gap's own
    rounding of 2^-24, times the exponent (at most 30) and ln 2: 2e-6 at the worst, for the last bit of gaps that are no fp32 numbers.  Weights are added as multiples of
    2^-(30 + leading zeros of V as a 32-bit number), 2^-50 for V = 3000, cut off below: every weight above 2^-50 (two here, those of -60 are nothing) by that much."""
    V = 3000
    for gap in (2.0, 8.0, 16.0, 20.0):
        logits = torch.full((1, V), -60.0)
        logits[0, 7], logits[0, 2000], logits[0, 2500] = gap, 0.0, 0.25
        for k, T in ((0, 1.0), (2, 1.0), (3, 0.7), (500, 1.3)):
            tok, lp = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")
            K.sample_rows_(logits.cuda(), tok, T, k, noise=torch.ones(V, device="cuda"), logprob_out=lp)
            want = drawn(logits[0].numpy(), np.float32(T), k, np.ones(V, dtype=np.float32))
            assert tok.item() == want[0] == 7
            rest = np.sort((logits[0].double().numpy() - gap) / float(np.float32(T)))[::-1][1 : k if k else V]
            exact = -np.log1p(np.exp(rest).sum())
            assert abs(lp.item() - exact) <= 2e-6 * abs(exact) + 2 * 2 ** -50, (gap, k, T, lp.item(), exact)


def test_draw_equal_logits(K):
    """Equal logits at the threshold are kept in the order of the tokens; of equal largest ones the lowest token."""
    V = 9000
    logits = torch.zeros(6, V)
    logits[:, [100, 8000]] = 2.0
    logits[:, 4000:] += torch.where(torch.arange(4000, V) % 7 == 0, 1.0, 0.0)
    logits[0] = -0.0
    logits[0, ::2] = 0.0       # no difference
    d = dict(logits=logits)
    for k in (1, 2, 3, 300, 716, 717, 718, 5000):
        e = exponential(6, V, seed=k)
        check_draw(K, d, 1.0, k, e)
        e = torch.full((6, V), 1e6)
        e[:, V - 1], e[:, 4004], e[:, 5] = 1e-6, 1e-5, 1e-4
        check_draw(K, d, 1.0, k, e)
    check_draw(K, d, 0.0, 4, None)


@pytest.mark.parametrize("V", [300, 9000, 40000])
@pytest.mark.parametrize("step", [None, 0.25, 2.0 ** -6])
def test_the_last_one_kept(K, V, step):
    """The k-th largest logit, equal ones in the order of their tokens, wins by its noise; the next one's noise is smaller still, but it is not kept.  step: logits are multiples of it."""
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(14, V, generator=g) * 2
    if step:
        logits = (logits / step).round() * step
    ks = [1, 2, 31, 100, 200, 255, 257, 299, 300, 500, 511, 512, 513, 1000]
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    e, want = torch.ones(14, V), []
    for b, k in enumerate(ks):
        k = min(k, V)
        want.append(order[b, k - 1].item())
        e[b, want[-1]] = 1e-20
        if k < V:
            e[b, order[b, k]] = 1e-30
    for l in (logits, logits.bfloat16()) if step else (logits,):
        if l.dtype == torch.bfloat16 and not torch.equal(l.float(), logits):
            continue
        tok = torch.zeros(14, dtype=torch.int64, device="cuda")
        K.sample_rows_(l.cuda(), tok, 1.0, torch.tensor(ks, dtype=torch.int32, device="cuda"), noise=e.cuda())
        assert tok.tolist() == want
        for b, k in enumerate(ks):    # a row at a time, by CTAs of other sizes
            K.sample_rows_(l[b : b + 1].cuda(), tok[:1], 1.0, k, noise=e[b : b + 1].cuda())
            assert tok[0].item() == want[b]


def test_draw_near_ties_go_by_64_bits(K):
    """Scores that 32 bits cannot tell apart."""
    V = 5000
    logits = torch.randn(3, V, generator=torch.Generator().manual_seed(3)) * 2
    e = exponential(3, V, seed=4)
    for b in range(3):
        score = (logits[b].double() - logits[b].double().max()) / 0.8 - e[b].double().log()
        best = score.argmax().item()
        for j, v in enumerate((17, 2500, 4999)):
            e[b, v] = torch.exp((logits[b, v].double() - logits[b].double().max()) / 0.8 - score[best]).float()
            if j == b:
                e[b, v] = torch.nextafter(e[b, v], torch.tensor(0.0))
    check_draw(K, dict(logits=logits), 0.8, None, e)


def test_draw_from_rows_that_leave_little(K):
    V = 3000
    d = dict(logits=torch.randn(6, V), ok=torch.zeros(6, V, dtype=torch.bool))
    d["ok"][1, 2999] = True
    d["ok"][2, [5, 6, 7]] = True
    d["logits"][3:] = float("nan")
    d["ok"][3:] = True
    d["logits"][4, 11] = -1e30
    d["logits"][5, 12], d["logits"][5, 13], d["logits"][5, 14] = float("inf"), 3.0, float("-inf")
    e = exponential(6, V)
    for k in (None, 1, 5, V):
        check_draw(K, d, 0.8, k, e)
        check_draw(K, d, 0.0, k, None)
    e[2, 6], e[2, 7], e[2, 5] = 0.0, float("inf"), 1e-40
    tok, _ = check_draw(K, dict(logits=d["logits"][:3], ok=d["ok"][:3]), 0.8, None, e[:3].clamp(max=3.4e38))
    assert tok.tolist() == [-1, 2999, 6]


@pytest.mark.parametrize("T", [1e-3, 1e-30, 1e4])
def test_draw_extreme_temperatures(K, T):
    d = make(4, 2000, counts=False, bias="", allowed="")
    check_draw(K, d, T, 100, exponential(4, 2000))


def test_settings_per_row_and_bookkeeping(K):
    B, V = 6, 4000
    d = make(B, V, torch.bfloat16, allowed="one", bias="one")
    T, k, e = torch.tensor([0.0, 0.5, 1.0, 1.5, 0.9, 0.0]), torch.tensor([5, 0, 1, 50, V, -3], dtype=torch.int32), exponential(V)
    want, _ = check_draw(K, d, T, k, e)
    for kind in (torch.int32, torch.int64):
        counts = d["counts"].cuda()
        pos, hist = torch.tensor([0, 3, 8, -1, -5, 9], device="cuda", dtype=kind), torch.full((B, 10), -7, device="cuda", dtype=kind)
        tok = torch.zeros(B, dtype=kind, device="cuda")
        kw = rules(K, d)
        kw["counts"] = counts
        K.sample_rows_(d["logits"].cuda(), tok, T.cuda(), k.cuda(), noise=e.cuda(), count=True, pos_inout=pos, history=hist, **kw)
        assert torch.equal(tok.long(), want) and pos.tolist() == [1, 4, 9, 0, -4, 10]
        more = d["counts"].clone()
        more[torch.arange(B), want.cpu()] += 1
        assert torch.equal(counts.cpu(), more)
        there = torch.full((B, 10), -7)
        for b, p in ((0, 1), (1, 4), (2, 9), (3, 0)):
            there[b, p] = want[b].item()
        assert torch.equal(hist.cpu().long(), there)
    for b in range(B):    # a row by itself
        tok = torch.zeros(1, dtype=torch.int64, device="cuda")
        kw = {n: (t[b : b + 1] if torch.is_tensor(t) and t.shape[0] == B else t) for n, t in rules(K, d).items()}
        K.sample_rows_(d["logits"][b : b + 1].cuda(), tok, T[b : b + 1].cuda(), k[b : b + 1].cuda(), noise=e.cuda(), **kw)
        assert tok.item() == want[b].item()


def test_random_states(K):
    """A row's Philox state: the same draws as the sampler of one row, whatever rows are beside it; captured draws go on from replay to replay."""
    V = 1000
    logits = torch.randn(3, V, generator=torch.Generator().manual_seed(5)).mul_(2).cuda()
    state = K.new_rng_state(torch.device("cuda"), seed=40, rows=3)
    assert state.tolist() == [[40, 0], [41, 0], [42, 0]]
    tok, hist, pos = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, 4001, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    run = lambda: K.sample_rows_(logits, tok, 0.9, 8, state, pos_inout=pos, history=hist)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3999):
        graph.replay()
    torch.cuda.synchronize()
    assert state[:, 1].tolist() == [4000] * 3 and pos.tolist() == [4000] * 3
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    for b in range(3):
        single = K.new_rng_state(torch.device("cuda"), seed=40 + b)
        for i in range(100):
            K.sample_(logits[b], one, 0.9, 8, single)
            assert one.item() == hist[b, i + 1].item()
        v, i = torch.topk(logits[b].cpu(), 8)
        p = torch.zeros(V)
        p[i] = torch.softmax(v / 0.9, -1)
        freq = torch.bincount(hist[b, 1:].cpu(), minlength=V) / 4000
        # 4000 draws: a frequency's standard deviation is at most 0.5 / sqrt(4000) = 0.008; five of them
        assert freq[p == 0].sum() == 0 and (freq - p).abs().max() < 0.04


@pytest.mark.parametrize("seed,token", [(207, 39758), (836, 28258), (909, 20637)])
def test_the_last_random_number_draws_nothing_by_itself(K, seed, token):
    """The states at whose offset 0 `token`'s 24 random bits are all ones: its u is rounded to 1, and an e of 0 would win over any logit.  Another token's lead of 40 is more than
    -ln of the smallest e (17.4) and ln of the largest (ln 17.4 = 2.9) together."""
    c, M = [token // 4, 0, 0, 0], 0xFFFFFFFF
    k0, k1 = seed, 0
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [b >> 32 ^ c[1] ^ k0, b & M, a >> 32 ^ c[3] ^ k1, a & M]
        k0, k1 = k0 + 0x9E3779B9 & M, k1 + 0xBB67AE85 & M
    assert c[token % 4] >> 8 == 0xFFFFFF
    logits = torch.zeros(2, 50257)
    logits[:, 11] = 40.0
    tok = torch.zeros(2, dtype=torch.int64, device="cuda")
    K.sample_rows_(logits.cuda(), tok, 1.0, None, torch.tensor([[seed, 0], [seed, 0]], device="cuda"))
    assert tok.tolist() == [11, 11]
    K.sample_rows_(logits.cuda(), tok, 1.0, 50256, torch.tensor([[seed, 0], [seed, 0]], device="cuda"))
    assert tok.tolist() == [11, 11]


def test_no_rows(K):
    empty = torch.empty(0, 50, device="cuda")
    assert K.adjust_logits(empty).shape == (0, 50)
    K.sample_rows_(empty, torch.empty(0, dtype=torch.int64, device="cuda"), 0.0)


def test_pack_allowed(K):
    for V in (1, 31, 32, 33, 100):
        ok = torch.rand(3, V) < 0.5
        words = K.pack_allowed(ok)
        assert words.dtype == torch.int32 and words.shape == (3, -(-V // 32))
        assert torch.equal(ok, torch.stack([(words[:, v // 32] >> (v % 32)) & 1 for v in range(V)], 1).bool())


def test_refusals(K):
    l = torch.zeros(3, 40, device="cuda")
    tok, i32 = torch.zeros(3, dtype=torch.int64, device="cuda"), lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    f = lambda *s: torch.zeros(*s, device="cuda")
    for kw in (dict(counts=f(3, 40)), dict(counts=i32(3, 39)), dict(counts=i32(40)), dict(bias=i32(40)), dict(bias=f(2, 40)), dict(allowed=i32(3, 3)), dict(allowed=f(2)),
               dict(repetition=0.0), dict(repetition=f(2)), dict(frequency=i32(3)), dict(bias=torch.zeros(40))):
        with pytest.raises(K.C.B200Error):
            K.adjust_logits(l, **kw)
        with pytest.raises(K.C.B200Error):
            K.sample_rows_(l, tok, 0.0, **kw)
    for bad in (l.half(), l[0], l.cpu()):
        with pytest.raises(K.C.B200Error):
            K.adjust_logits(bad)
    for out in (f(3, 39), f(3, 40).half(), f(40, 3).T):
        with pytest.raises(K.C.B200Error):
            K.adjust_logits(l, out=out)
    for args, kw in (((l, tok), {}), ((l, tok[:2], 0.0), {}), ((l, f(3), 0.0), {}), ((l, tok, f(2)), dict(noise=f(40))), ((l, tok, 1.0, f(3)), dict(noise=f(40))),
                     ((l, tok, 1.0), dict(noise=f(39))), ((l, tok, 1.0, None, torch.zeros(2, dtype=torch.int64, device="cuda")), {}), ((l, tok, 0.0), dict(count=True)),
                     ((l, tok, 0.0), dict(history=torch.zeros(3, 5, dtype=torch.int64, device="cuda"))), ((l, tok, 0.0), dict(pos_inout=i32(1))),
                     ((l, tok, 0.0), dict(logprob_out=f(2))), ((l, tok, 0.0), dict(pos_inout=i32(3), history=i32(3, 5)))):
        with pytest.raises(K.C.B200Error):
            K.sample_rows_(*args, **kw)
