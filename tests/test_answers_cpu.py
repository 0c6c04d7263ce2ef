"""Several answers to one prompt, what needs no GPU: refusals of the C entry points before any launch, the bookkeeping of forked and compacted requests."""
import ctypes
import struct

import pytest
import torch
import torch.nn as nn

from lit_gpt_b200 import _cabi as C
from lit_gpt_b200 import kernels as K
from lit_gpt_b200.generate.serve import Session
from lit_gpt_b200.ragged import SlotAllocator

FAKE = 0x10000   # never read: every call here is refused first


def refused(rc, text):
    assert rc == 1 and text in C.load().b200_last_error().decode(), (rc, C.load().b200_last_error())


def copies(tensors, slots, pairs):
    table = struct.pack("@" + "qqq" * len(tensors), *[v or 0 for t in tensors for v in t])
    pair = struct.pack("@" + "iiq" * len(pairs), *[v for p in pairs for v in p])
    return C.load().b200_copy_slots(table, len(tensors), slots, pair, len(pairs), None)


def test_copies_that_depend_on_each_other_are_refused():
    t = [(FAKE, 10, 64)]
    refused(copies(t, 4, [(0, 4, -1)]), "from slot 0 to 4 of 4")
    refused(copies(t, 4, [(-1, 2, -1)]), "from slot -1")
    refused(copies(t, 4, [(0, 1, -1), (1, 2, -1)]), "written by one copy and read by another")
    refused(copies(t, 4, [(2, 2, -1)]), "written by one copy and read by another")
    refused(copies(t, 4, [(0, 1, -1), (2, 1, -1)]), "written twice")
    refused(copies(t, 4, [(0, 1, 11)]), "11 positions")
    refused(copies([(None, 10, 64)], 4, [(0, 1, -1)]), "empty")
    refused(C.load().b200_copy_slots(None, 1, 4, None, 0, None), "null")
    assert copies(t, 4, []) == 0 and copies([], 4, [(0, 1, -1)]) == 0


def test_logit_rules_are_checked():
    lib = C.load()
    ok = dict(logits=FAKE, logits_dtype=C.F32, ld=8, rows=2, vocab=8, repetition_all=1.0)
    adjust = lambda out=FAKE, dtype=C.F32, apart=8, **kw: lib.b200_adjust_logits(ctypes.byref(C.LogitRules(**{**ok, **kw})), out, dtype, apart, None)
    refused(adjust(logits=None), "null")
    refused(adjust(logits_dtype=C.F16), "bf16 or fp32")
    refused(adjust(vocab=0), "0 logits")
    refused(adjust(vocab=1 << 30), "logits")
    refused(adjust(rows=-1), "-1 rows")
    refused(adjust(ld=-8), "distance")
    refused(adjust(out=None), "result")
    refused(adjust(dtype=C.F16), "result")
    refused(adjust(apart=7), "overlap")
    refused(adjust(dtype=C.BF16), "in place")
    refused(adjust(apart=16), "in place")
    refused(lib.b200_adjust_logits(None, FAKE, C.F32, 8, None), "null")
    draw = lambda **kw: lib.b200_sample_rows(ctypes.byref(C.LogitRules(**ok)), ctypes.byref(C.DrawArgs(**{**dict(token_out=FAKE, noise=FAKE), **kw})), None)
    refused(draw(token_out=None), "null")
    refused(draw(noise=None, temperature_all=0.5), "needs rng_state")
    refused(draw(noise=None, temperature=FAKE), "needs rng_state")
    refused(draw(count=1), "nothing to count")
    refused(draw(history=FAKE), "positions")
    refused(draw(noise_ld=-1), "distance")


def test_shared_prefix_arguments_are_checked():
    lib = C.load()
    ok = dict(qkv=FAKE, cos=FAKE, sin=FAKE, table_dtype=C.F32, table_rows=64, rope_n_elem=64, pos=FAKE, pos_count=1, k_cache=FAKE, v_cache=FAKE, k_batch_stride=2048,
              k_group_stride=1024, v_batch_stride=2048, v_group_stride=1024, k_prefix=FAKE, v_prefix=FAKE, k_prefix_stride=4096, v_prefix_stride=4096, out=FAKE, batch=3,
              n_head=4, n_groups=2, head_size=64, own_rows=16, prefix_rows=64, workspace=FAKE, workspace_bytes=1 << 30)
    call = lambda **kw: lib.b200_attn_decode_shared(ctypes.byref(C.AttnDecodeSharedArgs(**{**ok, **kw})), None)
    for kw, text in ((dict(head_size=80), "head size"), (dict(n_head=5), "heads"), (dict(batch=0), "batch"), (dict(own_rows=0), "lengths"), (dict(prefix_rows=-1), "lengths"),
                     (dict(qkv=None), "null"), (dict(k_prefix=None), "prefix"), (dict(rope_n_elem=66), "rope"), (dict(rope_n_elem=3), "rope"), (dict(cos=None), "tables"),
                     (dict(table_rows=0), "tables"), (dict(table_dtype=C.F16), "tables"), (dict(pos_count=2), "positions"), (dict(k_cache=FAKE + 2), "16-byte"),
                     (dict(v_prefix_stride=4100), "16-byte"), (dict(workspace_bytes=16), "workspace"), (dict(batch=1 << 23), "rows")):
        refused(call(**kw), text)
    refused(lib.b200_attn_decode_shared(None, None), "null")
    need = lib.b200_attn_decode_shared_workspace_bytes
    assert need(3, 4, 2, 64, 64, 16) > 0 and need(0, 4, 2, 64, 64, 16) == 0 and need(3, 4, 3, 64, 64, 16) == 0 and need(3, 4, 2, 80, 64, 16) == 0


def test_samples_need_the_gpu_cache():
    import lit_gpt_b200.generate.base as gb
    from lit_gpt_b200 import GPT, Config

    model = GPT(Config(name="t", block_size=32, vocab_size=50, padded_vocab_size=50, n_layer=1, n_head=2, n_embd=16))
    with pytest.raises(TypeError, match="set_kv_cache"):
        gb.generate_samples(model, torch.tensor([1, 2]), 8, 2)
    model.set_kv_cache(batch_size=1)
    with pytest.raises(NotImplementedError, match="GQA-native"):
        gb.generate_samples(model, torch.tensor([1, 2]), 8, 2)


@pytest.mark.parametrize("token", [-1, 50, 2 ** 40])
def test_prompts_that_are_counted_have_tokens_of_the_vocabulary(token):
    """A token outside has no place among the counts: refused on the host, before anything runs."""
    from types import SimpleNamespace

    import lit_gpt_b200.generate.base as gb
    from lit_gpt_b200 import GPT, Config
    from lit_gpt_b200.generate import serve

    model = GPT(Config(name="t", block_size=32, vocab_size=50, padded_vocab_size=50, n_layer=1, n_head=2, n_embd=16))
    model.set_kv_cache(batch_size=1)
    with pytest.raises(ValueError, match="outside 0 .. 49"):
        gb.generate_samples(model, torch.tensor([1, token]), 8, 2, presence_penalty=0.5, count_prompt=True)
    for kw in (dict(count_prompt=True), dict(presence_penalty=0.5)):    # nothing is counted in the prompt: as far as the refusal of this cache
        with pytest.raises(NotImplementedError, match="GQA-native"):
            gb.generate_samples(model, torch.tensor([1, token]), 8, 2, **kw)

    class Model(Slots):
        device, max_seq_length, config = torch.device("cpu"), 40, SimpleNamespace(vocab_size=50)

    model = Model(True)
    session = Session(model, slots=2)
    with pytest.raises(ValueError, match="outside 0 .. 49"):
        serve.generate_batch(model, [[1, 2], [4, token]], 3, session=session, presence_penalty=0.5, count_prompt=True)
    assert not session.live and (model.fed == -1).all()


def test_kept_steps_make_place_for_a_new_one(monkeypatch):
    """Where a step's caches find no place, the steps kept from earlier calls go first; where they find none even so, the call is refused."""
    import weakref

    import lit_gpt_b200.generate.base as gb

    class Step:
        full, asked = 0, []    # how many more find no place; how many steps were alive beside each

        def __init__(self, model, *key):
            Step.asked.append(sum(kept() is not None for kept in seen))
            if Step.full:
                Step.full -= 1
                raise torch.OutOfMemoryError("full")
            seen.append(weakref.ref(self))

    class Model:
        device = torch.device("cpu")

        def graph_key(self):
            return ("buffers",)

    monkeypatch.setattr(gb, "SampleGraph", Step)
    model, seen = Model(), []
    step = lambda rows: gb._sample_graph_for(model, rows, 64)
    assert step(16) is step(16) and Step.asked == [0]
    Step.full = 1
    assert step(3) is step(3) and Step.asked == [0, 1, 0] and len(model._sample_graphs) == 1
    Step.full = 2
    with pytest.raises(torch.OutOfMemoryError):
        step(5)
    assert Step.asked == [0, 1, 0, 1, 0] and not model._sample_graphs
    Step.full = 1
    with pytest.raises(torch.OutOfMemoryError):    # nothing was kept: not tried again
        step(5)
    assert Step.asked == [0, 1, 0, 1, 0, 0] and step(5) is step(5)


class Slots(nn.Module):
    """A model whose state of a slot is the tokens that it was fed."""

    def __init__(self, positional):
        super().__init__()
        self.positional_states, self.slots = positional, None

    def set_kv_cache(self, batch_size):
        self.fed, self.slots = torch.full((batch_size, 40, 1), -1), SlotAllocator(batch_size)

    def state_tensors(self):
        return [self.fed]

    def step(self, tokens, seqs, want):
        i = 0
        for slot, start, n in seqs:
            self.fed[slot, start : start + n, 0] = torch.tensor(tokens[i : i + n])
            i += n
        return torch.zeros(len(want), 1)


@pytest.mark.parametrize("positional", [True, False])
def test_fork_compact_and_shrink(monkeypatch, positional):
    def copy(tensors, src, dst, lengths=None):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst) and (lengths is not None) == positional
        for t in tensors:
            for i, (a, b) in enumerate(zip(src, dst)):
                n = t.shape[1] if lengths is None else lengths[i]
                t[b, :n] = t[a, :n]

    monkeypatch.setattr(K, "copy_slots", copy)
    model = Slots(positional)
    session = Session(model, slots=1)
    told = {}

    def feed(end=(), **tokens):
        session.step([(r, t, []) for r, t in tokens.items()], end=end)
        for r, t in tokens.items():
            told[r] = told.get(r, []) + t
        for r in end:
            del told[r]

    def check():
        assert set(session.live) == set(told) and len({s for s, _ in session.live.values()}) == len(told) == model.slots.in_use
        for r, (slot, n) in session.live.items():
            assert n == len(told[r]) and model.fed[slot, :n, 0].tolist() == told[r]

    feed(a=[1, 2, 3], b=[4])
    session.fork("a", ["c", "d", "e"])
    told.update({r: list(told["a"]) for r in "cde"})
    check()
    session.fork("b", [])
    feed(a=[5], c=[6, 7], d=[8], e=[9])
    feed(end=["a", "b", "d"], c=[10])
    check()
    session.compact()
    check()
    assert sorted(s for s, _ in session.live.values()) == [0, 1]
    feed(f=[11, 12])
    check()
    session.shrink()
    check()
    assert model.slots.capacity == 3
    feed(g=[13], c=[14])
    check()
    feed(end=["c", "e", "f", "g"])
    session.compact()
    session.shrink()
    check()
    assert model.slots.capacity == 1


@pytest.mark.parametrize("shape", [(39,), (41,), (1, 40), ()])
def test_a_grammar_speaks_about_every_token(monkeypatch, shape):
    """Truth values for more or fewer tokens than there are: refused, also where they pack into as many words."""
    from types import SimpleNamespace

    from lit_gpt_b200.generate import serve

    class Model(Slots):
        device, max_seq_length, config = torch.device("cpu"), 40, SimpleNamespace(vocab_size=40)

    drawn = []
    monkeypatch.setattr(K, "copy_slots", lambda *args: None)
    monkeypatch.setattr(K, "sample_rows_", lambda logits, token, *args, **kw: (drawn.append(kw["allowed"]), token.fill_(3)))
    model = Model(True)
    session = Session(model, slots=2)
    ask = lambda mask: serve.generate_batch(model, [[1, 2], [4]], 3, session=session, allowed=lambda i, tokens: mask)
    assert ask(torch.ones(40, dtype=torch.bool)) == [[1, 2, 3, 3, 3], [4, 3, 3, 3]] and all(w.shape == (2, 2) for w in drawn)
    drawn.clear()
    with pytest.raises(ValueError, match="40 tokens"):
        ask(torch.ones(shape, dtype=torch.bool))
    assert not drawn and not session.live
