"""Serving several requests over one model: the slot-managed cache, ragged steps, batched greedy / sampled generation, and
the replay of a recorded trace of steps.

``Session`` owns what a set of live requests needs: the model's caches (grown when more requests are live than there are
slots), one cache slot and the number of cached tokens per request.  ``Session.step`` is the one step function: every entry
brings the next tokens of a request, all entries run as one ragged batch (the model's ``step``), finished requests give their
slots back; the model is any that serves sequences from slots (``ragged.SlotServed`` with a ``step``).  ``generate_batch`` schedules prompts through it (prefill together, then one token per live request and step,
shorter requests leaving the batch early); ``Replayer`` feeds it recorded steps instead of sampled tokens.  ``PagedSession`` is the same for ``GPT`` models, over pages of one pool.
"""
from __future__ import annotations

import contextlib
from collections import Counter
from pathlib import Path
from typing import Any, Callable, Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from lit_gpt_b200 import kernels as K
from lit_gpt_b200.model import FUSED_HEAD_SIZES, GPT, PagedKVCache
from lit_gpt_b200.quant import weight_epoch
from lit_gpt_b200.ragged import PagedStep


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


class _Pages:
    """What a live request of a ``PagedSession`` holds."""

    __slots__ = ("pages", "cached", "position")

    def __init__(self) -> None:
        self.pages: List[int] = []   # its pages, in order
        self.cached = 0              # keys in them
        self.position = 0            # of its next token (more than `cached` once it has been cut down)


class _PagedGraph:
    """A captured decode step of up to `rows` requests with up to `width` pages each: one buffer carries the step's description and tokens to the device."""

    def __init__(self, session: "PagedSession", rows: int, width: int) -> None:
        self.rows, self.width = rows, width
        self.meta = torch.empty(rows * (7 + width), dtype=torch.int32, device=session.model.device)
        m = self.meta
        self.step = PagedStep(seqs=m[: 4 * rows].view(rows, 4), row_pos=m[4 * rows : 5 * rows], row_seq=m[5 * rows : 6 * rows], table=m[7 * rows :].view(rows, width), max_rows=1,
                              max_length=width * session.page)
        self.tokens = m[6 * rows : 7 * rows]
        self.fill([], [])   # requests that take no part: the warm-up leaves the caches as they are
        model = session.model
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                model.paged_step(self.tokens, self.step)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=session.graph_pool):
            self.logits = model.paged_step(self.tokens, self.step)
        self.graph = graph

    def fill(self, tokens: Sequence[int], requests: Sequence[_Pages]) -> None:
        n, rest = len(requests), self.rows - len(requests)
        host = torch.full((self.rows * (7 + self.width),), -1, dtype=torch.int32)
        seqs = [v for i, r in enumerate(requests) for v in (i, 1, r.cached, i)] + [0] * (4 * rest)
        host[: 7 * self.rows] = torch.tensor(seqs + [r.position for r in requests] + [0] * rest + list(range(n)) + [-1] * rest + list(tokens) + [0] * rest, dtype=torch.int32)
        table = host[7 * self.rows :].view(self.rows, self.width)
        for i, r in enumerate(requests):
            table[i, : len(r.pages)] = torch.tensor(r.pages, dtype=torch.int32)
        self.meta.copy_(host)


class PagedSession:
    """``Session`` for ``GPT`` models: the caches of all live requests are pages of one pool (``model.PagedKVCache``), taken as a request grows and given back when it ends, so that
    requests of any lengths share what memory there is.  ``step`` runs any mix of prompts, portions of prompts and single tokens as one ragged batch (``kernels.attn_paged``); steps of
    single tokens are captured and replayed.

    pages, page: how many pages the pool has, and keys of a page (16, 32, 64, 128 or 256).  keep: a request's cache is cut down to that many keys whenever it holds a page more, every group of
    heads by itself: the first `first` keys and the last `recent` stay, and of the others those that received most attention (``kernels.evict_paged``); positions go on.  portion: rows of
    one pass; longer prompts run in several, and are cut down between them: while one runs a request holds up to `portion` keys more.

    While a step runs the pool stands in the place of the model's own caches: one thread at a time works with a model, whether in its sessions or without."""

    GRAPHS = 8   # captured steps that are kept

    def __init__(self, model: Any, pages: int, page: int = 64, *, keep: Optional[int] = None, first: int = 4, recent: int = 64, portion: int = 4096) -> None:
        c = getattr(model, "config", None)
        if not isinstance(model, GPT) or model.device.type != "cuda" or model.transformer.wte.weight.dtype != torch.bfloat16 or c.head_size not in FUSED_HEAD_SIZES or c.rope_n_elem % 2 \
                or model.tp_world_size != 1 or model.spans_devices():
            raise NotImplementedError("a paged cache serves GPT models on one GPU in bf16, head size 64 or 128")
        if page not in (16, 32, 64, 128, 256) or pages < 1:
            raise ValueError(f"{pages} pages of {page} keys (16, 32, 64, 128 or 256)")
        if keep is not None and not (keep >= 1 and first >= 0 and recent >= 0 and first + recent <= keep):
            raise ValueError(f"{first} first and {recent} recent keys of {keep} to keep")
        if portion < 1:
            raise ValueError(f"a portion of {portion} rows")
        self.model, self.page, self.keep, self.first, self.recent, self.portion = model, page, keep, first, recent, portion
        self.caches = [PagedKVCache(c, pages, page, device=model.device, weights=keep is not None) for _ in model.transformer.h]
        self.live: Dict[Any, _Pages] = {}
        self._free = list(range(pages - 1, -1, -1))
        self._holders = [0] * pages   # requests that hold a page
        self.graph_pool = torch.cuda.graph_pool_handle()
        self._graphs: Dict[Tuple[int, int], _PagedGraph] = {}
        self._captured_for: Tuple = ()

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _tensors(self) -> List[torch.Tensor]:
        return [t for c in self.caches for t in (c.k, c.v, c.key_weights) if t is not None]

    def _take(self, request: _Pages, keys: int) -> None:
        """Pages for `keys` keys."""
        while len(request.pages) * self.page < keys:
            p = self._free.pop()
            self._holders[p] = 1
            request.pages.append(p)

    def _give(self, request: _Pages, keys: int = 0) -> None:
        """All pages behind those of the first `keys` keys."""
        left = -(-keys // self.page)
        for p in request.pages[left:]:
            self._holders[p] -= 1
            if self._holders[p] == 0:
                self._free.append(p)
        del request.pages[left:]

    @contextlib.contextmanager
    def _in_place(self):
        """The model over the pool."""
        blocks = self.model.transformer.h
        before = [b.attn.kv_cache for b in blocks]
        plan = self.model._fused_plan
        try:
            for b, cache in zip(blocks, self.caches):
                b.attn.kv_cache = cache
            self.model._fused_plan = None
            yield
        finally:
            for b, cache in zip(blocks, before):
                b.attn.kv_cache = cache
            self.model._fused_plan = plan

    def fork(self, rid: Any, new: Sequence[Any]) -> None:
        """Requests `new` that continue from where live request `rid` is.  Full pages are shared, the last one is copied for each (with `keep` all of them: what a key receives is
        each request's own)."""
        if rid not in self.live:
            raise KeyError(f"request {rid!r} is not live")
        new = list(new)
        if len(set(new)) != len(new) or any(n in self.live for n in new):
            raise ValueError("the requests of a fork are new ones, each of its own")
        source = self.live[rid]
        shared = source.cached // self.page if self.keep is None else 0
        used = -(-source.cached // self.page)
        if (used - shared) * len(new) > len(self._free):
            raise RuntimeError(f"{(used - shared) * len(new)} pages needed, {len(self._free)} of {len(self._holders)} are free")
        src, dst = [], []
        for n in new:
            r = _Pages()
            r.cached, r.position = source.cached, source.position
            r.pages = source.pages[:shared]
            for p in r.pages:
                self._holders[p] += 1
            self._take(r, source.cached)
            src += source.pages[shared:used]
            dst += r.pages[shared:]
            self.live[n] = r
        order = sorted(range(len(src)), key=lambda i: src[i])   # (neighbouring copies of one page read it once)
        K.copy_slots(self._tensors(), [src[i] for i in order], [dst[i] for i in order])

    def step(self, entries: Sequence[Tuple[Any, Sequence[int], Optional[Sequence[int]]]], end: Iterable[Any] = ()) -> Optional[torch.Tensor]:
        """As ``Session.step``: entries (request id, its next tokens, places among them whose logits are wanted or None for all); returns the wanted logits, fp32 (rows, vocab),
        in the order of the entries -- None when nothing is wanted.  Other than there an entry's rows come in the order of its tokens, whatever that of `places` is (a place that is
        named twice comes twice)."""
        K.raise_wait_errors()   # of the steps whose logits the caller has read since
        todo = [(rid, list(toks), Counter(range(len(toks)) if places is None else (int(p) for p in places))) for rid, toks, places in entries if toks]
        if len({rid for rid, _, _ in todo}) != len(todo):
            raise ValueError("a request has one entry in a step")
        need = 0
        for rid, toks, places in todo:
            r = self.live.get(rid)
            position, cached, held = (r.position, r.cached, len(r.pages)) if r is not None else (0, 0, 0)
            if position + len(toks) > self.model.max_seq_length:
                raise ValueError(f"request {rid!r}: position {position} and {len(toks)} tokens, max seq length is only {self.model.max_seq_length}")
            if min(toks) < 0 or max(toks) >= self.model.config.padded_vocab_size:
                raise ValueError(f"request {rid!r}: tokens outside 0 .. {self.model.config.padded_vocab_size - 1}")
            if any(not 0 <= p < len(toks) for p in places):
                raise ValueError(f"request {rid!r}: logits of places outside its {len(toks)} tokens are wanted")
            most = cached + len(toks) if self.keep is None else min(cached + len(toks), max(cached, self.keep + self.page) + self.portion)
            need += max(0, -(-most // self.page) - held)
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} of {len(self._holders)} are free")
        for rid, _, _ in todo:
            self.live.setdefault(rid, _Pages())
        done = [0] * len(todo)
        found: List[torch.Tensor] = []
        keys: List[Tuple[int, int]] = []   # (entry, place) of every row of `found`
        while any(done[i] < len(toks) for i, (_, toks, _) in enumerate(todo)):
            left, part = self.portion, []
            for i, (rid, toks, _) in enumerate(todo):
                n = min(left, len(toks) - done[i])
                if n > 0:
                    part.append((i, self.live[rid], toks[done[i] : done[i] + n]))
                    left -= n
            rows = [(i, done[i] + k) for i, _, toks in part for k in range(len(toks))]
            want = [k for k, (i, place) in enumerate(rows) for _ in range(todo[i][2][place])]
            for _, r, toks in part:
                self._take(r, r.cached + len(toks))
            logits = self._run([r for _, r, _ in part], [toks for _, _, toks in part], want)
            if want:
                found.append(logits)
                keys += [rows[k] for k in want]
            for i, r, toks in part:
                r.cached += len(toks)
                r.position += len(toks)
                done[i] += len(toks)
            if self.keep is not None:
                self._cut([r for _, r, _ in part if r.cached >= self.keep + self.page])
        for rid in end:
            r = self.live.pop(rid, None)
            if r is not None:
                self._give(r)
        if not found:
            return None
        logits = torch.cat(found) if len(found) > 1 else found[0]
        order = sorted(range(len(keys)), key=lambda k: keys[k])
        return (logits if order == list(range(len(keys))) else logits[torch.tensor(order, device=logits.device)]).float()

    def _run(self, requests: List[_Pages], tokens: List[List[int]], want: List[int]) -> Optional[torch.Tensor]:
        """One pass -> the wanted rows' logits."""
        dev = self.model.device
        with torch.inference_mode(), torch.cuda.device(dev), self._in_place():
            if all(len(t) == 1 for t in tokens):
                g = self._graph(len(requests), max(len(r.pages) for r in requests))
                g.fill([t[0] for t in tokens], requests)
                g.graph.replay()
                return g.logits[: len(requests)].clone() if want == list(range(len(requests))) else g.logits[torch.tensor(want, device=dev)] if want else None
            n, width = sum(len(t) for t in tokens), max(len(r.pages) for r in requests)
            seqs, row_seq, row_pos = [], [], []
            for i, (r, t) in enumerate(zip(requests, tokens)):
                seqs += [len(row_seq), len(t), r.cached, i]
                row_seq += [i] * len(t)
                row_pos += range(r.position, r.position + len(t))
            S, rows = len(requests), want if want else [n - 1]   # (without any wanted row the last one stands in)
            meta = torch.tensor(seqs + row_pos + row_seq + [t for part in tokens for t in part] + rows + [p for r in requests for p in r.pages + [-1] * (width - len(r.pages))],
                                dtype=torch.int32).to(dev, non_blocking=True)
            at = 4 * S
            step = PagedStep(seqs=meta[:at].view(S, 4), row_pos=meta[at : at + n], row_seq=meta[at + n : at + 2 * n], table=meta[at + 3 * n + len(rows) :].view(S, width),
                             max_rows=max(len(t) for t in tokens), max_length=max(r.cached + len(t) for r, t in zip(requests, tokens)))
            logits = self.model.paged_step(meta[at + 2 * n : at + 3 * n], step, meta[at + 3 * n : at + 3 * n + len(rows)])
            return logits if want else None

    def _graph(self, rows: int, width: int) -> _PagedGraph:
        """The captured step for that many requests and pages: up to the next of 1, 2, 4, 8, 16, 24, 32, .. requests, and pages in powers of two."""
        rows = 1 << (rows - 1).bit_length() if rows <= 16 else -(-rows // 8) * 8
        width = max(4, 1 << (width - 1).bit_length())
        model = self.model
        now = (model.max_seq_length, model.cos.data_ptr(), model.sin.data_ptr(), weight_epoch())   # what a captured step holds besides the pool
        if self._captured_for != now:
            self._graphs.clear()
            self._captured_for = now
        g = self._graphs.pop((rows, width), None)
        if g is None:
            while len(self._graphs) >= self.GRAPHS:
                self._graphs.pop(next(iter(self._graphs)))
            g = _PagedGraph(self, rows, width)
        self._graphs[(rows, width)] = g   # (the one used last stands last)
        return g

    def _cut(self, requests: List[_Pages]) -> None:
        """These requests' caches down to `keep` keys."""
        if not requests:
            return
        dev, width = self.model.device, max(len(r.pages) for r in requests)
        meta = torch.tensor([r.cached for r in requests] + [p for r in requests for p in r.pages + [-1] * (width - len(r.pages))], dtype=torch.int32).to(dev, non_blocking=True)
        lengths, table = meta[: len(requests)], meta[len(requests) :].view(len(requests), width)
        for c in self.caches:
            K.evict_paged(c.k, c.v, c.key_weights, table, lengths, self.keep, first=self.first, recent=self.recent, max_length=max(r.cached for r in requests))
        for r in requests:
            r.cached = self.keep
            self._give(r, self.keep)


def _session_for(model: Any, prompts: Sequence[Sequence[int]], max_new_tokens: int, num_samples: int) -> Any:
    """A session with room for these prompts and their answers."""
    if not isinstance(model, GPT):
        return Session(model, slots=len(prompts) * num_samples)
    page = 64
    pages = sum(-(-min(len(p) + max_new_tokens, model.max_seq_length) // page) for p in prompts) * num_samples
    return PagedSession(model, max(pages, 1), page)


@torch.inference_mode()
def generate_batch(model: Any, prompts: Sequence[Sequence[int]], max_new_tokens: int, *, temperature: float = 0.0, top_k: Optional[int] = None,
                   eos_id: Optional[int] = None, session: Optional[Union[Session, PagedSession]] = None, num_samples: int = 1, repetition_penalty: float = 1.0, frequency_penalty: float = 0.0,
                   presence_penalty: float = 0.0, count_prompt: bool = False, logit_bias: Optional[Dict[int, float]] = None,
                   allowed: Optional[Callable[[int, List[int]], Optional[torch.Tensor]]] = None) -> List[List[int]]:
    """Generate up to `max_new_tokens` tokens for each prompt, all prompts as one batch: one ragged prefill step, then one token
    per live request and step; a request that produced `eos_id` or reached the cache's length leaves the batch and frees its
    slot.  Returns prompt + generated ids per request.  temperature 0: greedy.  A ``GPT`` is served from a paged cache: without a `session` one with room for these
    prompts and answers, else a ``PagedSession`` of the caller's, which may hold less than they ask for where it cuts caches down.

    num_samples: that many answers to each prompt, which runs once and is forked (``Session.fork``); results then come prompt after prompt, num_samples each.
    Penalties count an answer's own tokens, with `count_prompt` its prompt's too (``kernels.adjust_logits``); logit_bias: token -> what is added to its logit;
    allowed: a grammar, called with a request's place in the results and its tokens so far, gives truth values (vocabulary,) of the tokens that may follow, or None
    for all; a request that it leaves none ends there."""
    from lit_gpt_b200.generate.base import _rng_for

    if num_samples < 1:
        raise ValueError(f"num_samples must be at least 1 (got {num_samples})")
    penalties = (float(repetition_penalty), float(frequency_penalty), float(presence_penalty))
    if num_samples > 1 or penalties != (1.0, 0.0, 0.0) or logit_bias or allowed is not None or isinstance(model, GPT):   # (all rows draw in one launch)
        session = session if session is not None else _session_for(model, prompts, max_new_tokens, num_samples)
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
                    session: Union[Session, PagedSession], num_samples: int, penalties: Tuple[float, float, float], count_prompt: bool, logit_bias: Optional[Dict[int, float]],
                    allowed: Optional[Callable[[int, List[int]], Optional[torch.Tensor]]]) -> List[List[int]]:
    """``generate_batch`` with several answers to a prompt or rules on the logits: all live requests draw in one launch and one host read per step."""
    from lit_gpt_b200.generate.base import row_rng_states

    dev, V, N = model.device, getattr(model.config, "padded_vocab_size", model.config.vocab_size), len(prompts) * num_samples
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
        if isinstance(model, GPT):
            K.check_gemv_errors(dev)


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
