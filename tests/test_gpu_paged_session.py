"""GPT models served from a paged cache through the public entry points: generate.serve.PagedSession and generate_batch."""
import dataclasses

import pytest
import torch

from test_gpu_answers import along, toy

pytestmark = pytest.mark.gpu


def prompts_of(n, vocab=500, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, vocab, (1 + (7 * i) % 41,), generator=g).tolist() for i in range(n)]


def follows(model, rc, pw, seq, T):
    l32, tol = along(model, rc, pw, torch.tensor(seq), T)
    chosen = l32.gather(1, torch.tensor(seq[T:])[:, None])[:, 0]
    assert (l32.amax(-1) - chosen <= 2 * tol).all()


@pytest.mark.parametrize("mode,name", [("nf4", "llama_gqa_hs64"), ("int4", "llama_mha_hs128"), (None, "llama_gqa_hs64")])
@pytest.mark.parametrize("n", [1, 3, 21])
@torch.inference_mode()
def test_greedy_batch_follows_the_oracle(golden, mode, name, n):
    """Prompts of unequal lengths as one batch, one token to more than the fused step's rows at a time."""
    from lit_gpt_b200.generate.serve import generate_batch

    model, rc, pw, _ = toy(golden, mode, name=name)
    assert model.fused_decode_ready() == (mode is not None)
    prompts = prompts_of(n)
    ys = generate_batch(model, prompts, 12)
    for p, y in zip(prompts, ys):
        assert y[: len(p)] == p and len(y) == len(p) + 12
    for p, y in list(zip(prompts, ys))[::4]:
        follows(model, rc, pw, y, len(p))
    assert model.transformer.h[0].attn.kv_cache.k.dim() == 4 and type(model.transformer.h[0].attn.kv_cache).__name__ == "KVCache"   # the model's own caches are where they were


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_logits_of_a_session(golden, mode):
    """Portions, wanted places, requests that come and go: every row's logits are the oracle's."""
    from lit_gpt_b200.generate.serve import PagedSession

    model, rc, pw, _ = toy(golden, mode)
    g = torch.Generator().manual_seed(3)
    seqs = {r: torch.randint(1, 500, (60,), generator=g) for r in "abcd"}
    want = {r: along(model, rc, pw, s, 1) for r, s in seqs.items()}      # logits behind every token but the last
    s = PagedSession(model, 24, 16, portion=25)
    at, rows = dict.fromkeys("abcd", 0), []

    def step(plan, end=()):
        entries = []
        for r, n, places in plan:
            entries.append((r, seqs[r][at[r] : at[r] + n].tolist(), places))
        logits = s.step(entries, end)
        k = 0
        for r, n, places in plan:
            for p in range(n) if places is None else sorted(places):
                l32, tol = want[r]
                assert (logits[k].cpu() - l32[at[r] + p]).abs().max() <= tol, (r, at[r] + p)
                k += 1
            at[r] += n
        assert (logits is None and k == 0) or logits.shape == (k, 512) and logits.dtype == torch.float32

    step([("a", 30, None), ("b", 1, None), ("c", 20, [19])])             # 51 rows: three passes of up to 25
    step([("b", 1, None), ("a", 1, None), ("c", 1, [])])
    step([("d", 9, [])])
    step([("d", 1, None), ("a", 3, [2, 0]), ("b", 17, [])], end=["c"])
    assert set(s.live) == set("abd") and [s.live[r].cached for r in "abd"] == [34, 19, 10]
    step([("a", 1, None), ("b", 1, None), ("d", 1, None)])
    step([("a", 20, [])], end=["a", "b", "d", "nobody"])
    assert s.free_pages == 24 and not s.live and not any(s._holders)


@torch.inference_mode()
def test_forks_share_full_pages(golden):
    from lit_gpt_b200.generate.serve import PagedSession

    model, rc, pw, _ = toy(golden)
    g = torch.Generator().manual_seed(4)
    head, tails = torch.randint(1, 500, (37,), generator=g).tolist(), torch.randint(1, 500, (3, 20), generator=g).tolist()
    for keep, pages in ((None, 3 + 2), (100, 3 + 6)):                    # two full pages and a part of one
        s = PagedSession(model, 40, 16, keep=keep, recent=8)
        s.step([("x", head, [])])
        s.fork("x", ["y", "z"])
        assert s.free_pages == 40 - pages
        for k in range(20):
            logits = s.step([(r, [t[k]], None) for r, t in zip("xyz", tails)])
        for r, t, row in zip("xyz", tails, logits.cpu()):
            l32, tol = along(model, rc, pw, torch.tensor(head + t + [0]), len(head) + 20)
            assert (row - l32[-1]).abs().max() <= tol
        with pytest.raises(KeyError):
            s.fork("nobody", ["w"])
        with pytest.raises(ValueError):
            s.fork("x", ["y"])
        with pytest.raises(RuntimeError, match="pages needed"):
            s.fork("x", [f"w{i}" for i in range(40)])
        s.step([], end="xyz")
        assert s.free_pages == 40


@torch.inference_mode()
def test_several_answers_and_rules(golden):
    from lit_gpt_b200.generate.serve import PagedSession, generate_batch

    model, rc, pw, prompt = toy(golden)
    prompts = [prompt.tolist(), prompt.tolist()[::-1] + [3]]
    ys = generate_batch(model, prompts, 15, num_samples=3, temperature=0.9)
    assert len(ys) == 6 and all(y[: len(prompts[i // 3])] == prompts[i // 3] and len(y) == len(prompts[i // 3]) + 15 for i, y in enumerate(ys))
    ys = generate_batch(model, prompts, 10, num_samples=2)
    assert ys[0] == ys[1] and ys[2] == ys[3]
    follows(model, rc, pw, ys[0], len(prompts[0]))
    for y in generate_batch(model, prompts, 30, temperature=0.7, presence_penalty=1e4):
        assert len(set(y[-30:])) == 30
    ok = torch.zeros(512, dtype=torch.bool)
    ok[[5, 9, 11]] = True
    s = PagedSession(model, 10, 16)
    ys = generate_batch(model, prompts, 8, temperature=1.0, session=s, allowed=lambda i, tokens: ok, eos_id=9)
    assert all(set(y[len(p) :]) <= {5, 9, 11} and 9 not in y[len(p) : -1] for p, y in zip(prompts, ys)) and s.free_pages == 10


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_caches_that_are_cut_down(golden, mode):
    """With room for all keys nothing changes; cut down, a request holds its first, its last and its heaviest keys, in order, goes on at its positions and gives its pages back."""
    from lit_gpt_b200.generate.serve import PagedSession

    model, rc, pw, _ = toy(golden, mode)
    g = torch.Generator().manual_seed(6)
    tokens = {r: torch.randint(1, 500, (150,), generator=g).tolist() for r in "ab"}

    def run(**kw):
        s = PagedSession(model, 40, 16, **kw)
        out = [s.step([("a", tokens["a"][:90], None), ("b", tokens["b"][:20], None)])]
        for k in range(60):
            out.append(s.step([("a", [tokens["a"][90 + k]], None), ("b", [tokens["b"][20 + k]], None)]))
        return s, torch.cat(out)

    # steps that record weights may run other kernels than those that do not: either side's logits are within `tol` of the oracle's, so within 2 tol of each other
    rc = dataclasses.replace(rc, block_size=200)
    tol = max(along(model, rc, pw, torch.tensor(t), 1)[1] for t in tokens.values())
    plain, want = run()
    same, got = run(keep=1000)
    assert (got - want).abs().max() <= 2 * tol and same.live["a"].cached == 150
    cut, got = run(keep=48, first=3, recent=10, portion=30)
    again, got2 = run(keep=48, first=3, recent=10, portion=30)
    assert torch.equal(got, got2) and torch.isfinite(got).all()
    assert (got[:30] - want[:30]).abs().max() <= 2 * tol   # (nothing had been cut yet)
    for r, n in (("a", 150), ("b", 80)):
        now = cut.live[r]
        assert now.position == n and 48 <= now.cached < 48 + 16 and len(now.pages) == -(-now.cached // 16)
    assert cut.free_pages == 40 - sum(len(x.pages) for x in cut.live.values())
    # the first layer's keys depend on token and position alone: which ones are left
    a, full = cut.live["a"], plain.live["a"]
    for group in range(model.config.n_query_groups):
        rows = lambda s, x: s.caches[0].k[torch.tensor(x.pages, device="cuda"), group].reshape(-1, 64)[: x.cached]
        match = (rows(cut, a)[:, None] == rows(plain, full)[None]).all(-1)
        assert match.sum(-1).eq(1).all()
        at = match.int().argmax(-1).tolist()
        since = a.cached - 48                                             # keys behind the last cut: all there, as are the ten before them
        assert at == sorted(at) and at[:3] == [0, 1, 2] and at[-since - 10 :] == list(range(150 - since - 10, 150))


@torch.inference_mode()
def test_refusals(golden):
    from lit_gpt_b200 import GPT, Config
    from lit_gpt_b200.generate.serve import PagedSession, generate_batch

    model, *_ = toy(golden)
    for kw in (dict(pages=0), dict(pages=4, page=48), dict(pages=4, keep=10, first=6, recent=5), dict(pages=4, keep=0), dict(pages=4, portion=0)):
        with pytest.raises(ValueError):
            PagedSession(model, **kw)
    with pytest.raises(NotImplementedError):
        PagedSession(GPT(Config(n_layer=1, n_head=2, n_embd=128, vocab_size=50, block_size=32)), 4)
    s = PagedSession(model, 4, 16)
    with pytest.raises(ValueError, match="max seq length"):
        s.step([("a", [1] * 201, None)])
    with pytest.raises(ValueError, match="one entry"):
        s.step([("a", [1], None), ("a", [2], None)])
    with pytest.raises(ValueError, match="places"):
        s.step([("a", [1, 2], [2])])
    with pytest.raises(RuntimeError, match="5 pages needed, 4 of 4 are free"):
        s.step([("a", [1] * 65, None)])
    assert not s.live and s.free_pages == 4
    s.step([("a", [1] * 60, [])])
    with pytest.raises(RuntimeError, match="pages needed"):
        generate_batch(model, [[1, 2, 3]], 80, session=s)
    assert list(s.live) == ["a"] and s.free_pages == 0
    assert s.step([], end=["a"]) is None and s.step([("a", [], None)]) is None
    assert model(torch.tensor([[1, 2]], device="cuda"), torch.arange(2, device="cuda")).shape[1] == 2   # the model's own caches are in place again
    with pytest.raises(TypeError, match="PagedKVCache"):
        model.paged_step(torch.tensor([1], device="cuda"), None)


@torch.inference_mode()
def test_tokens_outside_the_vocabulary_are_refused(golden):
    from lit_gpt_b200.generate.serve import PagedSession, generate_batch

    model, *_ = toy(golden)
    V = model.config.padded_vocab_size
    s = PagedSession(model, 8, 16)
    for bad in ([V], [1, -1], [3] * 20 + [1 << 40]):
        with pytest.raises(ValueError, match="tokens outside"):
            s.step([("a", [1, 2], None), ("b", bad, None)])
        with pytest.raises(ValueError, match="tokens outside"):
            generate_batch(model, [[1, 2], bad], 4)
    assert not s.live and s.free_pages == 8
    assert s.step([("a", [0, V - 1], None)]).shape == (2, V)
