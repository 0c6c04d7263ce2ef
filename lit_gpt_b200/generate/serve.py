"""Serving several requests over one model: the slot-managed cache, ragged steps, batched greedy / sampled generation, and
the replay of a recorded trace of steps.

``Session`` owns what a set of live requests needs: the model's caches (grown when more requests are live than there are
slots), one cache slot and the number of cached tokens per request.  ``Session.step`` is the one step function: every entry
brings the next tokens of a request, all entries run as one ragged batch (the model's ``step``), finished requests give their
slots back; the model is any that serves sequences from slots (``ragged.SlotServed`` with a ``step``).  ``generate_batch`` schedules prompts through it (prefill together, then one token per live request and step,
shorter requests leaving the batch early); ``Replayer`` feeds it recorded steps instead of sampled tokens.
"""
from __future__ import annotations

from pathlib import Path
from typing import Any, Callable, Dict, Iterable, List, Optional, Sequence, Tuple

import torch

from lit_gpt_b200 import kernels as K


class Session:
    def __init__(self, model: Any, slots: int = 4, max_seq_length: Optional[int] = None) -> None:
        self.model = model
        if max_seq_length is not None:
            model.max_seq_length = max_seq_length
        model.set_kv_cache(batch_size=max(1, slots))
        self.live: Dict[Any, List[int]] = {}    # request id -> [slot, cached tokens]

    def _grow(self) -> None:
        """Twice the slots, the live requests' caches and states carried over (slot numbers stay)."""
        model = self.model
        old = model.state_tensors()
        taken = {slot for slot, _ in self.live.values()}
        capacity = model.slots.capacity
        model.set_kv_cache(batch_size=2 * capacity)
        for new, prev in zip(model.state_tensors(), old):
            new[:capacity].copy_(prev)
        model.slots._free = [s for s in range(2 * capacity) if s not in taken]

    def _copy(self, src: Sequence[int], dst: Sequence[int], cached: Sequence[int]) -> None:
        K.copy_slots(self.model.state_tensors(), src, dst, list(cached) if self.model.positional_states else None)

    def fork(self, rid: Any, new: Sequence[Any]) -> None:
        """Requests `new` that continue from where live request `rid` is: its cached tokens and states are theirs too, each in a slot of its own."""
        if rid not in self.live:
            raise KeyError(f"request {rid!r} is not live")
        new = list(new)
        if len(set(new)) != len(new) or any(n in self.live for n in new):
            raise ValueError("the requests of a fork are new ones, each of its own")
        while self.model.slots.capacity - self.model.slots.in_use < len(new):
            self._grow()
        slot, cached = self.live[rid]
        slots = [self.model.slots.acquire() for _ in new]
        self._copy([slot] * len(new), slots, [cached] * len(new))
        for n, s in zip(new, slots):
            self.live[n] = [s, cached]

    def compact(self) -> None:
        """Moves live requests to the lowest slots: with n of them live, slots 0 .. n - 1 are theirs."""
        n = len(self.live)
        taken = {slot for slot, _ in self.live.values()}
        free = [s for s in range(n) if s not in taken]
        movers = sorted((state for state in self.live.values() if state[0] >= n), key=lambda state: state[0])
        self._copy([state[0] for state in movers], free, [state[1] for state in movers])
        for state, slot in zip(movers, free):
            state[0] = slot
        self.model.slots._free = list(range(n, self.model.slots.capacity))

    def shrink(self) -> None:
        """As many slots as requests are live (one at least), their caches and states carried over."""
        self.compact()
        model, n = self.model, max(1, len(self.live))
        old = model.state_tensors()
        model.set_kv_cache(batch_size=n)
        for new, prev in zip(model.state_tensors(), old):
            new.copy_(prev[:n])
        model.slots._free = list(range(len(self.live), n))

    def step(self, entries: Sequence[Tuple[Any, Sequence[int], Optional[Sequence[int]]]], end: Iterable[Any] = ()) -> Optional[torch.Tensor]:
        """entries: (request id, its next tokens, places among them whose logits are wanted or None for all).  Returns the
        wanted logits, fp32 (rows, vocab), in the order of the entries -- None when nothing is wanted."""
        K.raise_wait_errors()   # of the steps whose logits the caller has read since
        model = self.model
        tokens: List[int] = []
        seqs: List[Tuple[int, int, int]] = []
        want: List[int] = []
        for rid, toks, places in entries:
            if not toks:
                continue
            if rid not in self.live:
                if model.slots.in_use == model.slots.capacity:
                    self._grow()
                self.live[rid] = [model.slots.acquire(), 0]
            slot, cached = self.live[rid]
            places = range(len(toks)) if places is None else places
            want.extend(len(tokens) + int(p) for p in places)
            seqs.append((slot, cached, len(toks)))
            tokens.extend(int(t) for t in toks)
            self.live[rid][1] = cached + len(toks)
        logits = None
        if tokens:
            # rows nobody asks for still run (they fill the cache); without any wanted row the last one stands in and is dropped
            out = model.step(tokens, seqs, want if want else [len(tokens) - 1])
            logits = out if want else None
        for rid in end:
            state = self.live.pop(rid, None)
            if state is not None:
                model.slots.release(state[0])
        return logits


@torch.inference_mode()
def generate_batch(model: Any, prompts: Sequence[Sequence[int]], max_new_tokens: int, *, temperature: float = 0.0, top_k: Optional[int] = None,
                   eos_id: Optional[int] = None, session: Optional[Session] = None, num_samples: int = 1, repetition_penalty: float = 1.0, frequency_penalty: float = 0.0,
                   presence_penalty: float = 0.0, count_prompt: bool = False, logit_bias: Optional[Dict[int, float]] = None,
                   allowed: Optional[Callable[[int, List[int]], Optional[torch.Tensor]]] = None) -> List[List[int]]:
    """Generate up to `max_new_tokens` tokens for each prompt, all prompts as one batch: one ragged prefill step, then one token
    per live request and step; a request that produced `eos_id` or reached the cache's length leaves the batch and frees its
    slot.  Returns prompt + generated ids per request.  temperature 0: greedy.

    num_samples: that many answers to each prompt, which runs once and is forked (``Session.fork``); results then come prompt after prompt, num_samples each.
    Penalties count an answer's own tokens, with `count_prompt` its prompt's too (``kernels.adjust_logits``); logit_bias: token -> what is added to its logit;
    allowed: a grammar, called with a request's place in the results and its tokens so far, gives truth values (vocabulary,) of the tokens that may follow, or None
    for all; a request that it leaves none ends there."""
    from lit_gpt_b200.generate.base import _rng_for

    if num_samples < 1:
        raise ValueError(f"num_samples must be at least 1 (got {num_samples})")
    penalties = (float(repetition_penalty), float(frequency_penalty), float(presence_penalty))
    if num_samples > 1 or penalties != (1.0, 0.0, 0.0) or logit_bias or allowed is not None:
        session = session if session is not None else Session(model, slots=len(prompts) * num_samples)
        return _generate_ruled(model, prompts, max_new_tokens, temperature, top_k, eos_id, session, num_samples, penalties, count_prompt, logit_bias, allowed)
    session = session if session is not None else Session(model, slots=len(prompts))
    dev = model.device
    out = [list(p) for p in prompts]
    ids = [("gen", i) for i in range(len(prompts))]
    token = torch.empty(1, dtype=torch.int64, device=dev)
    rng = _rng_for(dev) if temperature > 0.0 else None

    def draw(logits: torch.Tensor) -> List[int]:
        picked = []
        for r in range(logits.shape[0]):
            K.sample_(logits[r : r + 1], token, temperature, top_k, rng)
            picked.append(int(token))
        K.raise_wait_errors()   # (the tokens were read back: the step is done)
        return picked

    live = list(range(len(prompts)))
    budget = [max_new_tokens] * len(prompts)
    nxt = draw(session.step([(ids[i], out[i], [len(out[i]) - 1]) for i in live])) if max_new_tokens > 0 else []
    while live:
        done = []
        for i, t in zip(live, nxt):
            out[i].append(t)
            budget[i] -= 1
            if budget[i] <= 0 or t == eos_id or len(out[i]) >= model.max_seq_length:
                done.append(i)
        live = [i for i in live if i not in done]
        if not live:
            session.step([], end=[ids[i] for i in done])
            break
        logits = session.step([(ids[i], [out[i][-1]], None) for i in live], end=[ids[i] for i in done])
        nxt = draw(logits)
    return out


def _generate_ruled(model: Any, prompts: Sequence[Sequence[int]], max_new_tokens: int, temperature: float, top_k: Optional[int], eos_id: Optional[int],
                    session: Session, num_samples: int, penalties: Tuple[float, float, float], count_prompt: bool, logit_bias: Optional[Dict[int, float]],
                    allowed: Optional[Callable[[int, List[int]], Optional[torch.Tensor]]]) -> List[List[int]]:
    """``generate_batch`` with several answers to a prompt or rules on the logits: all live requests draw in one launch and one host read per step."""
    from lit_gpt_b200.generate.base import row_rng_states

    dev, V, N = model.device, model.config.vocab_size, len(prompts) * num_samples
    out = [list(p) for p in prompts for _ in range(num_samples)]
    if N == 0 or max_new_tokens <= 0:
        return out
    if not all(out):
        raise ValueError("a prompt has one token at least")
    if logit_bias and not all(0 <= t < V for t in logit_bias):
        raise ValueError(f"logit_bias names tokens outside 0 .. {V - 1}")
    counted = penalties != (1.0, 0.0, 0.0)
    if counted and count_prompt and not all(0 <= t < V for p in prompts for t in p):
        raise ValueError(f"a prompt has tokens outside 0 .. {V - 1}, which cannot be counted")
    rng = row_rng_states(dev, N) if temperature > 0.0 else None
    counts = bias = None
    if counted:
        counts = torch.zeros(N, V, dtype=torch.int32, device=dev)
        if count_prompt:
            for i, p in enumerate(out):
                counts[i] = torch.bincount(torch.tensor(p, dtype=torch.int64, device=dev), minlength=V).int()
    if logit_bias:
        bias = torch.zeros(V, device=dev)
        bias[torch.tensor(list(logit_bias), device=dev)] = torch.tensor(list(logit_bias.values()), dtype=torch.float32, device=dev)

    def draw(logits: torch.Tensor, live: List[int]) -> List[int]:
        which = None if len(live) == N else torch.tensor(live, device=dev)
        words = None
        if allowed is not None:
            masks = [allowed(i, out[i]) for i in live]
            for i, m in zip(live, masks):
                if m is not None and m.shape != (V,):
                    raise ValueError(f"allowed gives truth values for {V} tokens (got {tuple(m.shape)} for request {i})")
            if any(m is not None for m in masks):
                words = K.pack_allowed(torch.stack([torch.ones(V, dtype=torch.bool) if m is None else m.to("cpu", torch.bool) for m in masks])).to(dev)
        token = torch.empty(len(live), dtype=torch.int64, device=dev)
        states, seen = (t if t is None or which is None else t[which] for t in (rng, counts))
        K.sample_rows_(logits, token, temperature, top_k, states, counts=seen, repetition=penalties[0], frequency=penalties[1], presence=penalties[2], bias=bias,
                       allowed=words, count=seen is not None)
        if which is not None:
            for t, part in ((rng, states), (counts, seen)):
                if t is not None:
                    t[which] = part
        picked = token.tolist()
        K.raise_wait_errors()   # (the tokens were read back: the step is done)
        return picked

    ids = [("gen", i) for i in range(N)]
    live, budget = list(range(N)), [max_new_tokens] * N
    try:
        first = session.step([(ids[p * num_samples], prompts[p], [len(prompts[p]) - 1]) for p in range(len(prompts))])
        for p in range(len(prompts)):
            session.fork(ids[p * num_samples], ids[p * num_samples + 1 : (p + 1) * num_samples])
        nxt = draw(first.repeat_interleave(num_samples, 0), live)
        while True:
            done = []
            for i, t in zip(live, nxt):
                if t >= 0:
                    out[i].append(t)
                budget[i] -= 1
                if t < 0 or budget[i] <= 0 or t == eos_id or len(out[i]) >= model.max_seq_length:
                    done.append(i)
            live = [i for i in live if i not in done]
            if not live:
                return out
            logits = session.step([(ids[i], [out[i][-1]], None) for i in live], end=[ids[i] for i in done])
            nxt = draw(logits, live)
    finally:
        session.step([], end=ids)   # (also when the grammar raises: the slots are the session's again)


class Replayer:
    """Feeds recorded steps ({"id", "tokens", "want"} entries, "end" lists) through a Session of the model in a directory."""

    def __init__(self, model_dir: Any, dtype: torch.dtype = torch.bfloat16, max_tokens: int = 0, device: Any = "cuda") -> None:
        from lit_gpt_b200.config import load_config, model_class

        config = load_config(Path(model_dir))
        cls = model_class(config)
        if not hasattr(cls, "step"):
            raise SystemExit(f"{cls.__name__} has no ragged step function: traces replay on models served through Session only")
        from lit_gpt_b200.checkpoint import load_registered

        self.model = load_registered(model_dir, dtype=dtype, device=device)
        bound = self.model.config.block_size
        if max_tokens and max_tokens < bound:
            # no request can be longer than what all live requests hold together: caches sized by position need no more than that
            self.model.max_seq_length = max_tokens
        slots = max(1, min(64, -(-max_tokens // self.model.max_seq_length))) if max_tokens else 2
        self.session = Session(self.model, slots=slots)

    def step(self, entries: Sequence[Dict[str, Any]], end: Iterable[Any] = ()) -> Optional[torch.Tensor]:
        return self.session.step([(e["id"], e.get("tokens", []), e.get("want", [])) for e in entries], end)
