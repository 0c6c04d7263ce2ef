"""Several answers to one prompt through the public entry points: generate.base.generate_samples (shared prefix, a draw per row), Session.fork / compact / shrink and
generate_batch with several samples and rules on the logits."""
import pytest
import torch

from oracle import model_ref as M

pytestmark = pytest.mark.gpu


def toy(golden, mode="nf4", max_seq=200, name="llama_gqa_hs64", batch=1):
    from test_gpu_model import build_cuda_model, cfg_from_golden, oracle_weights

    g = golden(name)
    cfgd, kw = cfg_from_golden(g)
    kw["block_size"] = max(kw["block_size"], max_seq)
    rc = M.RefConfig.from_any(cfgd)
    p = M.init_weights(rc, seed=1234)
    if mode is None:
        from lit_gpt_b200 import GPT, Config
        from lit_gpt_b200.fabric import Fabric

        fabric = Fabric(devices=1, precision="bf16-true")
        with fabric.init_module(empty_init=True):
            model = GPT(Config(**kw))
        with fabric.init_tensor():
            model.max_seq_length = max_seq
            model.set_kv_cache(batch_size=batch)
        model = fabric.setup_module(model.eval())
        model.load_state_dict({k: v.to(torch.bfloat16) for k, v in p.items()}, strict=True)
        pw = {k: v.to(torch.bfloat16).float() for k, v in p.items()}
    else:
        model, pw = build_cuda_model(kw, p, mode, max_seq, batch), oracle_weights(p, mode)
    return model, rc, pw, torch.from_numpy(g["gen_prompt"])


def along(model, rc, pw, seq, T):
    """The oracle's logits at the steps that chose seq[T:], and the tolerance of test_gpu_model.check_rollout."""
    from test_gpu_model import run_oracle

    cos, sin = model.cos.cpu(), model.sin.cpu()
    _, l32 = run_oracle(rc, pw, cos.float(), sin.float(), seq[:T], len(seq), torch.float32, forced=seq)
    _, l16 = run_oracle(rc, pw, cos, sin, seq[:T], len(seq), torch.bfloat16, forced=seq)
    return l32, 2.0 * (l16 - l32).abs().max().item() + 1e-3 * l32.abs().max().item()


@pytest.mark.parametrize("mode,name", [("nf4", "llama_gqa_hs64"), ("int4", "llama_mha_hs128"), (None, "llama_gqa_hs64")])
@torch.inference_mode()
def test_greedy_answers_follow_the_oracle(golden, mode, name):
    import lit_gpt_b200.generate.base as gb

    model, rc, pw, prompt = toy(golden, mode, name=name)
    assert model.fused_decode_ready() == (mode is not None)
    T = len(prompt)
    ys = gb.generate_samples(model, prompt.cuda(), T + 20, 19, temperature=0.0)    # two groups of rows where the step is fused
    assert len(ys) == 19 and all(torch.equal(y[:T].cpu(), prompt) and len(y) == T + 20 for y in ys)
    for y in {tuple(y.tolist()) for y in ys}:    # (rows of one group are the same numbers; groups of other sizes run other kernels)
        l32, tol = along(model, rc, pw, torch.tensor(y), T)
        chosen = l32.gather(1, torch.tensor(y[T:])[:, None])[:, 0]
        assert (l32.amax(-1) - chosen <= 2 * tol).all()
    assert len({tuple(y.tolist()) for y in ys[:16]}) == 1


@torch.inference_mode()
def test_drawn_answers_and_their_log_probabilities(golden):
    import lit_gpt_b200.generate.base as gb

    model, rc, pw, prompt = toy(golden)
    T = len(prompt)

    def answers(seed):
        torch.manual_seed(seed)
        gb._RNG.clear()
        return gb.generate_samples(model, prompt.cuda(), T + 30, 6, temperature=0.8, logprobs=True)

    ys, lps = answers(5)
    again, _ = answers(5)
    other, _ = answers(6)
    assert all(torch.equal(a, b) for a, b in zip(ys, again)) and not all(torch.equal(a, b) for a, b in zip(ys, other))
    assert len({tuple(y.tolist()) for y in ys}) == 6
    ys2 = gb.generate_samples(model, prompt.cuda(), T + 30, 6, temperature=0.8)    # the next call draws on
    assert not all(torch.equal(a, b) for a, b in zip(other, ys2))
    for y, lp in zip(ys, lps):
        l32, tol = along(model, rc, pw, y.cpu(), T)
        want = torch.log_softmax(l32 / 0.8, -1).gather(1, y[T:].cpu()[:, None])[:, 0]
        assert lp.shape == want.shape and ((lp.cpu() - want).abs() <= 2 * tol / 0.8).all()    # a logit off by tol moves its probability's logarithm by 2 tol / T at most


@torch.inference_mode()
def test_answers_end_at_eos_and_obey_their_rules(golden):
    import lit_gpt_b200.generate.base as gb

    model, rc, pw, prompt = toy(golden)
    T, p = len(prompt), prompt.cuda()
    ys = gb.generate_samples(model, p, T + 40, 9, temperature=1.0)
    eos = ys[0][T + 3].item()
    torch.manual_seed(3)
    for y in gb.generate_samples(model, p, T + 40, 9, temperature=1.0, eos_id=eos):
        body = y[T:].tolist()
        assert eos not in body[:-1] and (body[-1] == eos or len(body) == 40)
    for y in gb.generate_samples(model, p, T + 40, 5, temperature=0.7, frequency_penalty=1e4):
        assert len(set(y[T:].tolist())) == 40
    for y in gb.generate_samples(model, p, T + 40, 5, temperature=0.7, presence_penalty=1e4, count_prompt=True):
        assert len(set(y[T:].tolist())) == 40 and not set(y[T:].tolist()) & set(prompt.tolist())
    for y in gb.generate_samples(model, p, T + 20, 3, temperature=0.0, logit_bias={7: 1e6}):
        assert y[T:].tolist() == [7] * 20
    for y in gb.generate_samples(model, p, T + 20, 3, logit_bias={t: float("-inf") for t in range(50)}):
        assert min(y[T:].tolist()) >= 50
    one = gb.generate_samples(model, p, T + 1, 4, temperature=0.0)    # the first token alone
    assert len(one) == 4 and all(len(y) == T + 1 for y in one)


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_an_answer_ends_where_nothing_can_be_drawn(golden, mode):
    import lit_gpt_b200.generate.base as gb

    model, *_, prompt = toy(golden, mode)
    p, T = prompt.cuda(), len(prompt)
    nothing = {t: float("-inf") for t in range(model.config.padded_vocab_size)}
    ys, lps = gb.generate_samples(model, p, T + 12, 3, temperature=0.9, logit_bias=nothing, logprobs=True)
    assert all(torch.equal(y.cpu(), prompt) for y in ys) and all(lp.numel() == 0 for lp in lps)
    ys = gb.generate_samples(model, p, T + 12, 3, temperature=0.9, logit_bias=nothing, eos_id=5)
    assert all(torch.equal(y.cpu(), prompt) for y in ys)
    assert all(len(y) == T + 12 for y in gb.generate_samples(model, p, T + 12, 3, temperature=0.9))


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_answers_that_can_draw_nothing_end_the_steps(golden, mode, monkeypatch):
    """Rows that ended without a token count as ended where an eos_id is looked for: the steps stop at the next look."""
    import lit_gpt_b200.generate.base as gb

    model, *_, prompt = toy(golden, mode)
    p, T, V = prompt.cuda(), len(prompt), model.config.padded_vocab_size
    steps, step = [], gb.SampleGraph.step
    monkeypatch.setattr(gb.SampleGraph, "step", lambda self: (steps.append(1), step(self))[1])
    nothing = {t: float("-inf") for t in range(V)}
    ys = gb.generate_samples(model, p, T + 100, 3, temperature=0.9, logit_bias=nothing, eos_id=5)
    assert all(torch.equal(y, p) for y in ys) and len(steps) == gb.EOS_POLL
    # two tokens may follow, each once: an answer holds both, or ends with the one that ends it
    steps.clear()
    two = {t: float("-inf") for t in range(V) if t not in (7, 9)}
    for y in gb.generate_samples(model, p, T + 100, 6, temperature=1.5, logit_bias=two, presence_penalty=float("inf"), eos_id=8):
        assert sorted(y[T:].tolist()) == [7, 9]
    assert len(steps) == gb.EOS_POLL
    steps.clear()
    for y in gb.generate_samples(model, p, T + 100, 6, temperature=1.5, logit_bias=two, presence_penalty=float("inf"), eos_id=9):
        assert y[T:].tolist() in ([9], [7, 9])
    assert len(steps) == gb.EOS_POLL


@pytest.mark.parametrize("draw", ["sample_rows_", "argmax_", "sample_"])
@torch.inference_mode()
def test_a_capture_that_fails_leaves_no_graph(golden, monkeypatch, draw):
    """An exception behind most of a captured step's launches (of several answers, of one, of a prompt): the next call captures anew and does not replay what there is of it."""
    import lit_gpt_b200.generate.base as gb

    model, *_, prompt = toy(golden)
    first, then = prompt.cuda()[:8], prompt.flip(0).cuda()[:8]
    call = (lambda p: gb.generate_samples(model, p, 28, 3, temperature=0.0)) if draw == "sample_rows_" else lambda p: [gb.generate(model, p, 28, temperature=0.0)]
    want = call(then)
    model.set_kv_cache(batch_size=1, device="cuda", dtype=torch.bfloat16)    # (lets the captured steps go)
    whole = getattr(gb.K, draw)

    def fails(*args, **kw):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("no more")
        return whole(*args, **kw)

    with monkeypatch.context() as m:
        m.setattr(gb.K, draw, fails)
        with pytest.raises(RuntimeError, match="no more"):
            call(first)
    assert all(torch.equal(a, b) for a, b in zip(call(then), want))


@torch.inference_mode()
def test_one_captured_step_serves_prompts_of_all_lengths(golden):
    import lit_gpt_b200.generate.base as gb

    model, *_ = toy(golden)
    fresh, *_ = toy(golden)
    g = torch.Generator().manual_seed(8)
    alone = torch.randint(0, 100, (11,), generator=g).cuda()
    before = gb.generate(model, alone, 40, temperature=0.0)
    for T in (9, 60, 3, 100):
        prompt = torch.randint(0, 100, (T,), generator=g).cuda()
        ys = gb.generate_samples(model, prompt, T + 25, 4, temperature=0.0)
        fresh.__dict__.pop("_sample_graphs", None)
        for blk in fresh.transformer.h:
            blk.attn.kv_cache.reset_parameters()
        assert all(torch.equal(a, b) for a, b in zip(ys, gb.generate_samples(fresh, prompt, T + 25, 4, temperature=0.0)))
    assert len(model._sample_graphs) == 1 and next(iter(model._sample_graphs.values())).graph is not None
    assert torch.equal(before, gb.generate(model, alone, 40, temperature=0.0))    # the model's own caches and captured step
    model.max_seq_length = 150
    model.set_kv_cache(batch_size=2, device="cuda", dtype=torch.bfloat16)
    assert "_sample_graphs" not in model.__dict__
    ys = gb.generate_samples(model, alone, 40, 3, temperature=0.0)
    assert all(torch.equal(ys[0], y) for y in ys)


@torch.inference_mode()
def test_refusals(golden):
    import lit_gpt_b200.generate.base as gb

    model, _, _, prompt = toy(golden)
    p, T = prompt.cuda(), len(prompt)
    for kw, error in ((dict(num_samples=0), ValueError), (dict(num_samples=2, logit_bias={-1: 1.0}), ValueError), (dict(num_samples=2, logit_bias={10 ** 6: 1.0}), ValueError)):
        with pytest.raises(error):
            gb.generate_samples(model, p, T + 5, **kw)
    with pytest.raises(NotImplementedError):
        gb.generate_samples(model, p, 1000, 2)
    sg = gb._sample_graph_for(model, 2, 64, 0.0, None, (1.0, 0.0, 0.0), False, False, p.dtype)
    with sg.in_place(), pytest.raises(RuntimeError, match="one token each"):
        model(p.view(1, -1).expand(2, -1).contiguous(), torch.arange(T, device="cuda"))
    model.clear_kv_cache()
    with pytest.raises(TypeError):
        gb.generate_samples(model, p, T + 5, 2)


@torch.inference_mode()
def test_traced_step_over_a_shared_prefix(golden):
    import torch._dynamo

    import lit_gpt_b200.generate.base as gb

    model, _, _, prompt = toy(golden)
    p, T = prompt.cuda(), len(prompt)
    model(p.view(1, -1), torch.arange(T, device="cuda"))
    sg = gb._sample_graph_for(model, 3, 64, 0.0, None, (1.0, 0.0, 0.0), False, False, p.dtype)
    sg.prefix_len.fill_(T)
    tok, pos = torch.tensor([[1], [2], [3]], device="cuda"), torch.tensor([T], device="cuda")
    with sg.in_place():
        want = model(tok, pos).float()
        torch._dynamo.reset()
        with torch.inference_mode(False), torch.no_grad():
            got = torch.compile(model, backend="eager", fullgraph=True)(tok, pos).float()
    # another order of the same roundings to bf16 (norms and products are not fused): the rounding points differ by a few steps of 2^-8
    assert (got - want).abs().max() <= 2 ** -5 * want.abs().max()


# ---- models that serve sequences from slots -----------------------------------------------------------------------------------------
def _kinds():
    import test_gpu_fizadra as F
    import test_gpu_fovirax as X
    import test_gpu_lefalix as L
    import test_gpu_nulezen as N
    import test_gpu_pomipel as P
    import test_gpu_votavik as V

    return {"lefalix": (L, L.CFG_ODD, {}), "pomipel": (P, P.CFG_ODD, dict(max_seq=200)), "fizadra": (F, F.CFG_ODD, dict(max_seq=200)), "nulezen": (N, N.CFG_ODD, {}),
            "votavik": (V, V.CFG_ODD, {}), "fovirax": (X, X.CFG_ODD, {})}


@pytest.mark.parametrize("kind", ["lefalix", "pomipel", "fizadra", "nulezen", "votavik", "fovirax"])
def test_forked_requests_go_their_own_ways(kind):
    from lit_gpt_b200.generate.serve import Session

    mod, cfg, kw = _kinds()[kind]
    w = mod.checkpoint(cfg, 21)
    model = mod.build(cfg, w, torch.float32, slots=2, **kw)
    session = Session(model, slots=2)
    prompt, other = mod.tokens_for(cfg, 23, 1), mod.tokens_for(cfg, 9, 2)
    session.step([("p", prompt, []), ("q", other, [])])
    session.fork("p", ["a", "b", "c"])                   # grows
    assert model.slots.in_use == 5 and session.live["b"][1] == 23
    with pytest.raises(KeyError):
        session.fork("nobody", ["x"])
    for new in (["a"], ["x", "x"], ["q"]):
        with pytest.raises(ValueError):
            session.fork("p", new)
    follow = {r: mod.tokens_for(cfg, 12, 30 + i) for i, r in enumerate("pabcq")}
    seq = {r: (other if r == "q" else prompt) + follow[r] for r in follow}
    alone = {r: mod.O.forward(cfg[0] if isinstance(cfg, tuple) else cfg, w, t) for r, t in seq.items()}
    start = {r: len(seq[r]) - 12 for r in seq}

    def steps(live, first, last, end=()):
        for i in range(first, last):
            out = session.step([(r, [follow[r][i]], [0]) for r in live], end=end if i == last - 1 else ())
            for j, r in enumerate(live):
                assert mod.rel_err(out[j], alone[r][start[r] + i]) < 1e-4, (r, i)

    steps("pabcq", 0, 4, end=["p", "b"])
    session.compact()
    assert sorted(s for s, _ in session.live.values()) == [0, 1, 2] and model.slots.in_use == 3
    steps("acq", 4, 7)
    session.shrink()
    assert model.slots.capacity == 3 and model.slots.in_use == 3
    steps("acq", 7, 9, end=["q"])
    session.fork("a", ["d"])
    follow["d"], alone["d"], start["d"] = follow["a"], alone["a"], start["a"]
    steps("acd", 9, 12)
    session.step([], end=["a", "c", "d"])
    session.shrink()
    assert model.slots.capacity == 1 and model.slots.in_use == 0


@pytest.mark.parametrize("kind", ["lefalix", "pomipel"])
def test_batches_of_samples_and_rules(kind):
    import lit_gpt_b200.generate.base as gb
    from lit_gpt_b200.generate.serve import Session, generate_batch

    mod, cfg, kw = _kinds()[kind]
    model = mod.build(cfg, mod.checkpoint(cfg, 22), torch.float32, **kw)
    V = cfg["vocab"]
    prompts = [mod.tokens_for(cfg, 9, 3), mod.tokens_for(cfg, 4, 4)]
    plain = generate_batch(model, prompts, 11)
    ys = generate_batch(model, prompts, 11, num_samples=3)
    assert ys == [plain[0]] * 3 + [plain[1]] * 3 and model.slots.in_use == 0
    session = Session(model, slots=1)

    def drawn(seed):
        torch.manual_seed(seed)
        gb._RNG.clear()
        return generate_batch(model, prompts, 11, num_samples=4, temperature=1.0, top_k=30, session=session)

    a, b = drawn(1), drawn(1)
    assert a == b and a != drawn(2) and len({tuple(y) for y in a}) == 8 and not session.live
    eos = a[0][len(prompts[0]) + 2]
    for y, p in zip(generate_batch(model, prompts, 30, num_samples=4, temperature=1.0, eos_id=eos), [prompts[0]] * 4 + [prompts[1]] * 4):
        assert y[: len(p)] == p and eos not in y[len(p) : -1] and (y[-1] == eos or len(y) == len(p) + 30)
    for y, p in zip(generate_batch(model, prompts, 30, temperature=0.5, presence_penalty=1e4, count_prompt=True, num_samples=2), [prompts[0]] * 2 + [prompts[1]] * 2):
        assert len(set(y)) == len(set(p)) + 30
    even = torch.arange(V) % 2 == 0
    calls = []

    def grammar(i, tokens):
        calls.append((i, len(tokens)))
        if i == 1 and len(tokens) == len(prompts[1]) + 5:
            return torch.zeros(V, dtype=torch.bool)
        return even if i == 0 else None

    y0, y1 = generate_batch(model, prompts, 11, allowed=grammar)
    assert len(y0) == 20 and all(t % 2 == 0 for t in y0[9:]) and len(y1) == 9 and y1 == plain[1][:9] and (0, 9) in calls
    assert generate_batch(model, prompts, 5, logit_bias={3: 1e6})[0][9:] == [3] * 5
    with pytest.raises(ValueError):
        generate_batch(model, prompts, 5, logit_bias={V: 1.0})
    assert generate_batch(model, [], 5, num_samples=2) == [] and generate_batch(model, prompts, 0, num_samples=2) == [prompts[0]] * 2 + [prompts[1]] * 2

    def broken(i, tokens):
        if len(tokens) == len(prompts[i // 2]) + 3:
            raise RuntimeError("no such rule")

    with pytest.raises(RuntimeError, match="no such rule"):
        generate_batch(model, prompts, 8, num_samples=2, allowed=broken, session=session)
    assert not session.live and model.slots.in_use == 0
    assert generate_batch(model, prompts, 8, num_samples=2, session=session) == [plain[0][:17]] * 2 + [plain[1][:12]] * 2
    with pytest.raises(ValueError, match="one token at least"):
        generate_batch(model, [[], prompts[0]], 5, num_samples=2, session=session)
    assert not session.live


# ---- the command line ---------------------------------------------------------------------------------------------------------------
def command(directory, *args):
    import pathlib
    import subprocess
    import sys

    root = pathlib.Path(__file__).resolve().parent.parent
    res = subprocess.run([sys.executable, "-m", "lit_gpt_b200.generate.base", *args, "--checkpoint_dir", str(directory)], cwd=root, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-2000:]
    return res.stdout.strip().splitlines(), res.stderr


@pytest.mark.parametrize("quantize", [["--quantize", "bnb.nf4"], []])
def test_command_line(tmp_path, golden, quantize):
    """Answers as a batch from a checkpoint directory with a tokenizer, whose prompts are 32-bit tokens."""
    import json

    from tokenizers import Tokenizer, models, pre_tokenizers
    from test_gpu_model import cfg_from_golden

    from lit_gpt_b200 import Config

    cfgd, kw = cfg_from_golden(golden("llama_gqa_hs64"))
    kw["block_size"] = max(kw["block_size"], 128)
    V = Config(**kw).padded_vocab_size
    torch.save({k: v.to(torch.bfloat16) for k, v in M.init_weights(M.RefConfig.from_any(cfgd), seed=1234).items()}, tmp_path / "lit_model.pth")
    (tmp_path / "lit_config.json").write_text(json.dumps(kw))
    words = Tokenizer(models.WordLevel({f"t{i}": i for i in range(V)}, unk_token="t0"))
    words.pre_tokenizer = pre_tokenizers.WhitespaceSplit()
    words.save(str(tmp_path / "tokenizer.json"))
    (tmp_path / "tokenizer_config.json").write_text("{}")
    prompt = [f"t{i}" for i in (5, 17, 3, 88, 41, 7)]
    ask = lambda *args: command(tmp_path, " ".join(prompt), "--max_new_tokens", "30", *quantize, *args)
    plain, _ = ask("--temperature", "0")
    lines, said = ask("--temperature", "0", "--num_samples", "5", "--batch_samples", "true")
    assert len(lines) == 5 and len(set(lines)) == 1 and "Time for inference of 5" in said
    assert lines[0].split()[:7] == plain[0].split()[:7] and len(lines[0].split()) == len(plain[0].split()) == 36
    lines, _ = ask("--num_samples", "3", "--presence_penalty", "10000")
    assert len(set(lines)) == 3
    for line in lines:
        assert line.split()[:6] == prompt and len(line.split()) == 36 and len(set(line.split()[6:])) == 30


def test_command_line_of_a_slot_served_model(tmp_path):
    import test_gpu_fizadra as F

    w = F.checkpoint(F.CFG_ODD, 111)
    F._write_checkpoint(tmp_path, F.CFG_ODD, w)
    prompt = F.tokens_for(F.CFG_ODD, 6, 112)
    want = F.O.greedy(F.CFG_ODD, w, prompt, 9)
    lines, _ = command(tmp_path, " ".join(map(str, prompt)), "--precision", "32-true", "--temperature", "0", "--max_new_tokens", "9", "--num_samples", "3", "--batch_samples", "true")
    assert [list(map(int, line.split())) for line in lines] == [want] * 3
    lines, _ = command(tmp_path, " ".join(map(str, prompt)), "--precision", "32-true", "--max_new_tokens", "20", "--frequency_penalty", "10000")
    assert len(lines) == 1 and len(set(lines[0].split()[6:])) == 20 and len(lines[0].split()) == 26


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_prompts_of_32_bit_tokens(golden, mode):
    import lit_gpt_b200.generate.base as gb

    model, *_, prompt = toy(golden, mode)
    T = len(prompt)
    kw = dict(temperature=0.0, presence_penalty=2.0, count_prompt=True, logprobs=True, eos_id=3)
    want, scores = gb.generate_samples(model, prompt.long().cuda(), T + 20, 3, **kw)
    got, scores32 = gb.generate_samples(model, prompt.int().cuda(), T + 20, 3, **kw)
    assert all(a.dtype == torch.int32 and torch.equal(a.long(), b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(scores32, scores))


@torch.inference_mode()
def test_the_last_group_of_rows_takes_the_place_of_the_others(golden, monkeypatch):
    """A last, smaller group of rows whose caches find no place beside the step of the groups before: that one is let go."""
    import weakref

    import lit_gpt_b200.generate.base as gb

    model, *_, prompt = toy(golden)
    p, T = prompt.cuda(), len(prompt)
    want = gb.generate_samples(model, p, T + 20, 19, temperature=0.0)
    model.__dict__.pop("_sample_graphs")
    there = []

    class Step(gb.SampleGraph):
        def __init__(self, model, *key):
            if any(step() is not None for step in there):
                raise torch.OutOfMemoryError("full")
            super().__init__(model, *key)
            there.append(weakref.ref(self))

    monkeypatch.setattr(gb, "SampleGraph", Step)
    got = gb.generate_samples(model, p, T + 20, 19, temperature=0.0)
    assert len(got) == 19 and all(torch.equal(a, b) for a, b in zip(got, want)) and [step() is None for step in there] == [True, False]
