"""Continuous-batching step loop over the paged int8 cache: scheduler, page pool and CUDA-graph replay around
the attention ops.

It plays the role of kbwal/inference-engine qwen3-1.7b/engine.py for this library's paged cache:

* the same public surface (`submit_request`, `step`, `generate`, a `Request` with prompt, output and times)
  and the same scheduling policy (engine.py:143-204): every decoding request gets its token first, then
  requests in the middle of their prompt continue, then waiting requests are admitted first come first served
  while the step's token budget lasts; a prompt's first chunk is at least `min_first_chunk` tokens (or the
  whole prompt);
* the same bookkeeping (engine.py:229-252): a request produces its first token when the last chunk of its
  prompt is in the cache, and ends on the stop token, on `max_new_tokens`, or when the cache row is full;
* the same execution scheme (engine.py:376-470): pure-decode steps replay one CUDA graph per batch-size bucket,
  steps with prefill one graph per token bucket, all inputs of a step travel in one int32 buffer at fixed
  addresses, and a step that fits no bucket runs eagerly.

What differs is the cache: the reference gives every request a cache row of `max_len` tokens (a slot); here
the cache is a pool of 16-token pages and a request holds a list of them.  `PagePool` hands pages out on
demand (append on decode, release on finish); a request is admitted only if the pages its whole lifetime can
need are still uncommitted, so a running request can never run out.  The first pages of the pool are a
scratch run no request owns: padded entries of a graph replay write there.

A model whose layers carry a state from token to token (`stateful`) also gets one state slot per request: taken when the
request is admitted, given back when it ends, and never cleared, since a request at position 0 starts from zero.  Padded
entries have slot -1, which the recurrent kernels pass over.

`Scheduler` is host-only (no torch, no GPU) so that the policy is testable on its own; `Engine` adds the
device side.  It drives any model of the registry (models/__init__.py): the model makes its own caches and runs one
step; sampling is the library's Gumbel-max sampler (greedy at tau = 0).  Besides generating (`submit_request`, `step`),
the engine replays given tokens (`open_replay`, `replay`, `close_replay`) through the same step, cache and graphs and
hands out the logits of any of them.

Requests may bring things of their own, if the engine is made for that: a way of sampling with penalties, biases and a grammar
(`own_sampling`; `Sampling`), and a low-rank adapter out of the model's slots (`adapters`).  Both travel in the step's input buffer, so
the same graphs serve whatever the requests ask for; without them steps are what they were.
"""
from __future__ import annotations

import math
import time
import traceback
from collections import deque
from collections.abc import Callable
from dataclasses import dataclass, field


MOST_FLOAT, LEAST_FLOAT = (2 - 2.0 ** -23) * 2.0 ** 127, 2.0 ** -126  # of 32 bits


@dataclass(frozen=True)
class Sampling:
    """How one request's tokens are chosen (ops.Draw, ops.Rules): by default the most likely one.  bias: token -> what is added to its logit.
    grammar: called with the output so far, returns the row of the engine's masks for the next token, -1: none; if it raises or there is no such
    row, the request ends with that error.  seed: of the request's random numbers (default: the engine's and the request's number)."""

    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: dict[int, float] = field(default_factory=dict)
    grammar: Callable[[list[int]], int] | None = None
    seed: int | None = None

    def __post_init__(self):
        numbers = (self.temperature, self.top_p, self.min_p, self.repetition, self.presence, self.frequency, *self.bias.values())
        if not all(abs(x) <= MOST_FLOAT for x in numbers):
            raise ValueError("sampling: a number is none, or infinite in 32 bits")
        if (self.temperature < 0 or not 0 <= self.top_k < 2 ** 31 or not 0 < self.top_p <= 1 or not 0 <= self.min_p <= 1
                or self.repetition < LEAST_FLOAT or (self.seed is not None and self.seed < 0)):
            raise ValueError(f"sampling: {self} is out of range")


@dataclass
class Request:
    id: int
    prompt_ids: list[int]
    max_new_tokens: int
    pages: list[int] = field(default_factory=list)  # physical pages, in token order
    slot: int = -1  # state slot, for models that carry a state
    committed: int = 0  # pages promised to this request at admission and not yet handed out
    cached_len: int = 0  # tokens currently in the cache
    output: list[int] = field(default_factory=list)
    sampling: Sampling | None = None
    adapter: int = -1
    history: int = -1  # row of the engine's token histories, for requests with a way of sampling
    rng: object = None
    error: Exception | None = None  # what its grammar ended it with
    admitted: bool = False
    t_submit: float = 0.0
    t_first_token: float | None = None
    t_finish: float | None = None

    @property
    def decoding(self) -> bool:
        return self.cached_len >= len(self.prompt_ids)


def without_frames(e: Exception) -> Exception:
    """The exception with its traceback as text: the frames would keep the engine, its cache and its graphs alive as long as the request."""
    e.add_note("".join(traceback.format_exception(e)))
    at = e
    while at is not None:
        at.__traceback__ = None
        at = at.__cause__ or at.__context__
    return e


class PagePool:
    """Free list of physical pages [first, num_pages).  `commit` promises pages without choosing them,
    `take` turns one promise into a page, `release` returns pages and drops leftover promises."""

    def __init__(self, num_pages: int, first: int = 0):
        self.free = list(range(num_pages - 1, first - 1, -1))  # pop() hands out the lowest id first
        self.committed = 0
        self.capacity = num_pages - first

    def uncommitted(self) -> int:
        return len(self.free) - self.committed

    def commit(self, n: int) -> bool:
        if n > self.uncommitted():
            return False
        self.committed += n
        return True

    def take(self) -> int:
        assert self.committed > 0 and self.free
        self.committed -= 1
        return self.free.pop()

    def release(self, pages: list[int], leftover_promises: int = 0) -> None:
        assert leftover_promises <= self.committed
        self.committed -= leftover_promises
        self.free.extend(sorted(pages, reverse=True))


class SlotPool:
    """State slots 0 .. n - 1, the lowest free one first."""

    def __init__(self, n: int):
        self.free = list(range(n - 1, -1, -1))
        self.capacity = n

    def take(self) -> int:
        if not self.free:
            raise RuntimeError("every state slot is in use")
        return self.free.pop()

    def release(self, slot: int) -> None:
        if slot >= 0:
            self.free.append(slot)
            self.free.sort(reverse=True)


@dataclass
class Step:
    entries: list[tuple[Request, list[int]]]  # decoding requests first (one token each), then prefill chunks
    num_decoding: int
    masks: dict[int, int] = field(default_factory=dict)  # request id -> the mask that its grammar asks for

    @property
    def decode_only(self) -> bool:
        return self.num_decoding == len(self.entries)

    @property
    def num_tokens(self) -> int:
        return sum(len(t) for _, t in self.entries)


class Scheduler:
    def __init__(self, max_batch_size: int, max_len: int, page_size: int, pool: PagePool, max_tokens_per_step: int,
                 min_first_chunk: int, stop_token_id: int, slots: SlotPool | None = None, histories: SlotPool | None = None):
        assert max_tokens_per_step >= max_batch_size + min_first_chunk, \
            "the budget must fit every decoding request plus one first chunk, or prefill can stall forever"
        self.max_batch_size, self.max_len, self.page_size = max_batch_size, max_len, page_size
        self.pool, self.max_tokens_per_step, self.min_first_chunk = pool, max_tokens_per_step, min_first_chunk
        self.stop_token_id, self.slots, self.histories = stop_token_id, slots, histories
        self.running: list[Request] = []
        self.waiting: deque[Request] = deque()
        self.next_id = 0

    def submit(self, prompt_ids: list[int], max_new_tokens: int) -> Request:
        assert max_new_tokens >= 1 and len(prompt_ids) > 0
        assert len(prompt_ids) + max_new_tokens <= self.max_len, "prompt + continuation must fit max_len"
        need = math.ceil(min(len(prompt_ids) + max_new_tokens - 1, self.max_len) / self.page_size)
        if need > self.pool.capacity:  # it could never be admitted and would block the queue for ever
            raise ValueError(f"the request needs {need} pages over its lifetime, the pool holds {self.pool.capacity}")
        r = Request(self.next_id, list(prompt_ids), max_new_tokens, t_submit=time.perf_counter())
        self.next_id += 1
        self.waiting.append(r)
        return r

    def idle(self) -> bool:
        return not self.running and not self.waiting

    def lifetime_pages(self, r: Request) -> int:
        # the last generated token is never written to the cache
        return math.ceil(min(len(r.prompt_ids) + r.max_new_tokens - 1, self.max_len) / self.page_size)

    def plan(self) -> Step | None:
        budget = self.max_tokens_per_step
        entries: list[tuple[Request, list[int]]] = []
        for r in self.running:  # decoding requests are never starved and come first
            if r.decoding:
                entries.append((r, [r.output[-1]]))
                budget -= 1
        num_decoding = len(entries)
        for r in self.running:  # requests in the middle of their prompt
            if not r.decoding and budget > 0:
                n = min(len(r.prompt_ids) - r.cached_len, budget)
                entries.append((r, r.prompt_ids[r.cached_len : r.cached_len + n]))
                budget -= n
        while self.waiting and len(self.running) < self.max_batch_size and budget > 0:
            r = self.waiting[0]
            if self.slots is not None and not self.slots.free:
                break
            n = min(len(r.prompt_ids), budget)
            if n < min(len(r.prompt_ids), self.min_first_chunk):
                break  # first come first served: nobody overtakes it
            if not self.pool.commit(self.lifetime_pages(r)):
                break  # the pool cannot promise its whole lifetime yet
            self.waiting.popleft()
            r.committed, r.admitted = self.lifetime_pages(r), True
            if self.slots is not None:
                r.slot = self.slots.take()
            if self.histories is not None:
                r.history = self.histories.take()
            self.running.append(r)
            entries.append((r, r.prompt_ids[:n]))
            budget -= n
        if not entries:
            return None
        for r, toks in entries:  # pages for the tokens this step writes
            need = math.ceil((r.cached_len + len(toks)) / self.page_size) - len(r.pages)
            for _ in range(need):
                r.pages.append(self.pool.take())
                r.committed -= 1
        return Step(entries, num_decoding)

    def commit(self, step: Step, sampled: list[int]) -> list[Request]:
        now = time.perf_counter()
        finished = []
        for (r, toks), tok in zip(step.entries, sampled):
            r.cached_len += len(toks)
            if r.decoding:
                none = tok < 0 and self.histories is not None  # its rules allow no token: the request ends
                if not none:
                    r.output.append(int(tok))
                    if len(r.output) == 1:
                        r.t_first_token = now
                if none or tok == self.stop_token_id or len(r.output) >= r.max_new_tokens or r.cached_len + 1 >= self.max_len:
                    self.end(r, now)
                    finished.append(r)
        return finished

    def end(self, r: Request, now: float) -> None:
        self.pool.release(r.pages, r.committed)
        r.pages, r.committed = [], 0
        if self.histories is not None:
            self.histories.release(r.history)
            r.history = -1
        if self.slots is not None:
            self.slots.release(r.slot)
            r.slot = -1
        self.running.remove(r)
        r.t_finish = now


class Engine:
    """Scheduler + device execution.  `model`: an instance of a registered model class on a CUDA device.  `num_slots`: state
    slots of a stateful model, one per live request (default: one per request of the largest batch).  `own_sampling`: requests may have a
    Sampling of their own (the others are drawn at the temperature tau, as in engines without), of up to `max_bias` biased tokens, under grammars of
    up to `num_masks` masks (set_mask).  `adapters`: requests may name a slot of the model's adapters (model.make_adapters before, and not again)."""

    slots: SlotPool | None = None
    # what an entry's sampling comes to on the device, an array each, int32 and then fp32
    SAMPLING_INTS = ("slots", "lengths", "prompts", "mask_rows", "top_k")
    SAMPLING_FLOATS = ("repetition", "presence", "frequency", "temperature", "top_p", "min_p", "uniform")

    def __init__(self, model, max_batch_size: int, max_len: int, stop_token_id: int, page_size: int | None = None,
                 num_pages: int | None = None, max_tokens_per_step: int = 1024, min_first_chunk: int = 64,
                 max_graph_tokens: int = 512, use_graphs: bool = True, block_m: int = 128, tau: float = 0.0, seed: int = 0,
                 num_slots: int | None = None, own_sampling: bool = False, max_bias: int = 16, num_masks: int = 64, adapters: bool = False):
        import numpy as np
        import torch

        from . import kernels as K
        from . import scaffold as S

        self.torch, self.K, self.S, self.np = torch, K, S, np
        self.model, self.device = model, model.device
        page_size = model.page_size if page_size is None else page_size
        model.tau = float(tau)  # baked into the graphs at capture, like the reference's (engine.py:399)
        model.seed.fill_(seed)
        self.page_size, self.max_len, self.block_m = page_size, max_len, block_m
        self.max_batch_size = max_batch_size
        self.num_entries = max_batch_size + 1  # every request plus one padding entry
        self.max_pages = math.ceil(max_len / page_size)  # block-table width
        # token buckets of steps with prefill (engine.py:254-259) and batch buckets of pure-decode steps
        M = min(max_graph_tokens, max_tokens_per_step, max_len)
        self.token_buckets = sorted({b for b in (16, 32, 64) if b < M} | set(range(128, M, 128)) | {M})
        self.graph_buckets = sorted({min(1 << i, max_batch_size) for i in range(max_batch_size.bit_length() + 1)})
        # scratch run: the padding entry of the largest bucket writes that many tokens from position 0
        self.scratch_pages = math.ceil(max(self.token_buckets) / page_size)
        assert self.scratch_pages <= self.max_pages
        if num_pages is None:  # what the reference's slot rows hold: max_len tokens per request
            num_pages = self.scratch_pages + max_batch_size * self.max_pages
        self.pool = PagePool(num_pages, first=self.scratch_pages)
        if getattr(model, "stateful", False):
            self.slots = SlotPool(max_batch_size if num_slots is None else num_slots)
        self.own_sampling, self.max_bias, self.seed, self.tau = own_sampling, max_bias, seed, float(tau)
        self.adapter_slots, self.adapters = 0, None
        if adapters:
            if getattr(model, "adapters", None) is None:
                raise ValueError("the model has no slots for adapters: make_adapters comes first")
            self.adapters = model.adapters  # (the recorded steps read these)
            self.adapter_slots = next(iter(model.adapters[0].values())).slots
        if own_sampling:
            if max_bias < 0 or num_masks < 1:
                raise ValueError("own_sampling needs room for a mask, and not less than none for biases")
            self.history = torch.zeros(max_batch_size, max_len, dtype=torch.int32, device=self.device)
            self.masks = torch.full((num_masks, (model.vocab + 31) // 32), -1, dtype=torch.int32, device=self.device)
        self.sched = Scheduler(max_batch_size, max_len, page_size, self.pool, max_tokens_per_step, min_first_chunk,
                               stop_token_id, self.slots, SlotPool(max_batch_size) if own_sampling else None)
        per_slot = {} if self.slots is None else {"slots": self.slots.capacity}
        self.caches = model.make_caches(num_pages, page_size, self.max_pages * page_size, **per_slot)
        # one int32 buffer per kind of step, filled on the host and copied in one piece
        cap = sum(self.mixed_layout(max_tokens_per_step))
        self.host_mixed = torch.empty(cap, dtype=torch.int32).pin_memory()
        self.dev_mixed = torch.zeros(cap, dtype=torch.int32, device=self.device)
        capd = sum(self.decode_layout())
        self.host_decode = torch.empty(capd, dtype=torch.int32).pin_memory()
        self.dev_decode = torch.zeros(capd, dtype=torch.int32, device=self.device)
        self.np_mixed, self.np_decode = self.host_mixed.numpy(), self.host_decode.numpy()  # same memory
        self.rows: dict[int, tuple] = {}  # request id -> (pages copied so far, its block-table row as an array)
        self.scratch_row = self.np.zeros(self.max_pages, self.np.int32)
        self.scratch_row[: self.scratch_pages] = self.np.arange(self.scratch_pages)
        self.prefix_capacity = 2 * max_len
        self.prefix = model.make_prefix(self.prefix_capacity)  # None: the model reads its cache by page
        self.graph_pool = torch.cuda.graph_pool_handle()  # one pool for all graphs: only one runs at a time
        self.decode_graphs: dict[int, tuple] = {}
        self.mixed_graphs: dict[int, tuple] = {}
        self.steps_run = {"decode_graph": 0, "mixed_graph": 0, "eager": 0}
        self.seconds = {"plan": 0.0, "run (inputs, launch, read-back)": 0.0, "commit": 0.0, "inputs": 0.0}
        if use_graphs:
            self.capture()

    # ------------------------------------------------------------------ public surface (engine.py:120-142)
    def submit_request(self, prompt_ids: list[int], max_new_tokens: int, sampling: Sampling | None = None, adapter: int = -1) -> Request:
        if sampling is not None:
            if not self.own_sampling:
                raise ValueError("the engine was made without own_sampling")
            if len(sampling.bias) > self.max_bias or any(not 0 <= t < self.model.vocab for t in sampling.bias):
                raise ValueError(f"up to {self.max_bias} biased tokens of 0 .. {self.model.vocab - 1} are wanted")
        if adapter != -1 and not 0 <= adapter < self.adapter_slots:
            raise ValueError(f"adapter {adapter}: the engine has {self.adapter_slots} slots")
        if self.own_sampling and any(not 0 <= t < self.model.vocab for t in prompt_ids):
            raise ValueError(f"a prompt has ids outside 0 .. {self.model.vocab - 1}")
        r = self.sched.submit(prompt_ids, max_new_tokens)
        if sampling is None and self.own_sampling and self.tau > 0:
            sampling = Sampling(self.tau)
        r.sampling, r.adapter = sampling, adapter
        if self.own_sampling:
            s = sampling.seed if sampling is not None else None
            r.rng = self.np.random.default_rng([self.seed % 2 ** 64, r.id] if s is None else s)
        return r

    def set_mask(self, row: int, allowed) -> None:
        """Mask `row` allows these token ids and no others (in stream order: steps that run already keep the one before)."""
        if not self.own_sampling or not 0 <= row < self.masks.shape[0]:
            raise ValueError(f"mask {row}: the engine has {self.masks.shape[0] if self.own_sampling else 0}")
        bits = self.np.zeros(self.masks.shape[1] * 32, self.np.uint8)
        ids = self.np.asarray(list(allowed), self.np.int64)
        if ids.size and (ids.min() < 0 or ids.max() >= self.model.vocab):
            raise ValueError(f"a token id outside 0 .. {self.model.vocab - 1}")
        bits[ids] = 1
        words = self.np.packbits(bits, bitorder="little").view(self.np.int32)
        self.masks[row].copy_(self.torch.from_numpy(words))

    def generate(self, prompts: list[list[int]], max_new_tokens: int, sampling: Sampling | None = None, adapter: int = -1) -> list[Request]:
        reqs = [self.submit_request(p, max_new_tokens, sampling, adapter) for p in prompts]
        while not self.sched.idle():
            self.step()
        return reqs

    def step(self) -> list[Request]:
        t0 = time.perf_counter()
        step = self.sched.plan()
        if step is None:
            return []
        finished = self.ask_grammars(step)
        t1 = time.perf_counter()
        tokens = self.run(step).tokens[: len(step.entries)].tolist() if step.entries else []  # the read-back ends the step
        t2 = time.perf_counter()
        finished += self.sched.commit(step, tokens)
        for r in finished:
            self.rows.pop(r.id, None)
        self.seconds["plan"] += t1 - t0
        self.seconds["run (inputs, launch, read-back)"] += t2 - t1
        self.seconds["commit"] += time.perf_counter() - t2
        return finished

    # ------------------------------------------------------------------ replay of given tokens
    def open_replay(self) -> Request:
        """A request whose tokens the caller supplies; it holds pages like any other."""
        r = Request(self.sched.next_id, [], 0, admitted=True)
        self.sched.next_id += 1
        return r

    def replay(self, entries: list[tuple[Request, list[int], list[int]]]):
        """One step of (request, its next tokens, places among them whose logits are wanted).  Returns the wanted
        logits, fp32 [wanted, vocab], in the order of the entries; the tokens the step samples are dropped."""
        for r, toks, want in entries:
            if not toks or r.cached_len + len(toks) > self.max_len:
                raise ValueError(f"{r.cached_len} + {len(toks)} tokens do not fit a request of {self.max_len}")
            if any(not 0 <= t < self.model.vocab for t in toks) or any(not 0 <= w < len(toks) for w in want):
                raise ValueError("a token id or a wanted place is out of range")
        # decoding entries (one token behind cached ones) come first, as in the steps the scheduler plans
        order = sorted(range(len(entries)), key=lambda i: not (len(entries[i][1]) == 1 and entries[i][0].cached_len > 0))
        decoding = sum(len(toks) == 1 and r.cached_len > 0 for r, toks, _ in entries)
        for r, toks, _ in entries:
            need = math.ceil((r.cached_len + len(toks)) / self.page_size) - len(r.pages)
            if not self.pool.commit(need):
                raise RuntimeError("the page pool is exhausted")
            r.pages.extend(self.pool.take() for _ in range(need))
            if self.slots is not None and r.slot < 0:
                r.slot = self.slots.take()
        step = Step([entries[i][:2] for i in order], decoding)
        out = self.run(step)
        first, at = {}, 0
        for i in order:
            first[i] = at
            at += len(entries[i][1])
        rows = [first[i] + w for i, (_, _, want) in enumerate(entries) for w in want]
        for r, toks, _ in entries:
            r.cached_len += len(toks)
        with self.torch.inference_mode():
            if not rows:
                return self.torch.empty(0, self.model.vocab)
            return self.model.logits(out.hidden[self.torch.tensor(rows, device=self.device)]).float().cpu()

    def close_replay(self, r: Request) -> None:
        self.pool.release(r.pages)
        r.pages = []
        if self.slots is not None:
            self.slots.release(r.slot)
            r.slot = -1
        self.rows.pop(r.id, None)

    # ------------------------------------------------------------------ input buffers
    def step_entries(self, n_tokens: int, live: int | None = None) -> int:
        """Entries of a step with prefill, the padding one included: for a bucket as many as its tokens can belong to, for a step
        that is not recorded those it has (`live`; above eight in steps of eight, since decode attention keeps a workspace
        for each number).  The kernels choose their forms, and lay out their grids, by this number."""
        if live is None:
            return min(self.num_entries, n_tokens + 1)
        return min(self.num_entries, live + 1 if live < 8 else -(-(live + 1) // 8) * 8)

    def mixed_layout(self, n_tokens: int, live: int | None = None) -> list[int]:
        """Field lengths of a step with prefill padded to n_tokens: ids, positions, seq_ids, cu_seqlens,
        cached_lens, cu_cached, tile_start, num_decoding, block table, state slots, and what the requests ask.  The same n_tokens always
        gives a bucket the same layout, so its fields always sit at the same addresses."""
        E = self.step_entries(n_tokens, live)
        return [n_tokens, n_tokens, n_tokens, E + 1, E, E + 1, math.ceil(n_tokens / self.block_m) + E, 1, E * self.max_pages, E,
                self.asks_size(E, n_tokens)]

    def asks_size(self, entries: int, rows: int) -> int:
        """Adapters of the rows; then, per entry, the sampling fields and the biases (tokens, values)."""
        n = rows if self.adapter_slots else 0
        if self.own_sampling:
            n += (len(self.SAMPLING_INTS) + len(self.SAMPLING_FLOATS) + 2 * self.max_bias) * entries
        return n

    def wants_token(self, r: Request, toks: list[int]) -> bool:
        return r.history >= 0 and r.cached_len + len(toks) >= len(r.prompt_ids)

    def mask_of(self, r: Request) -> int:
        grammar = None if r.sampling is None else r.sampling.grammar
        mask = -1 if grammar is None else int(grammar(r.output))
        if not -1 <= mask < self.masks.shape[0]:
            raise ValueError(f"request {r.id}: its grammar asks for mask {mask} of {self.masks.shape[0]}")
        return mask

    def ask_grammars(self, step: Step) -> list[Request]:
        """The masks of the step's requests, before anything of it is done: a request whose grammar fails ends, and the others have their step."""
        failed = []
        for r, toks in step.entries if self.own_sampling else ():
            if r.sampling is None or r.sampling.grammar is None or not self.wants_token(r, toks):
                continue
            try:
                step.masks[r.id] = self.mask_of(r)
            except Exception as e:
                r.error = without_frames(e)
                failed.append(r)
        for r in failed:
            at = next(i for i, (q, _) in enumerate(step.entries) if q is r)
            step.num_decoding -= at < step.num_decoding
            del step.entries[at]
            self.sched.end(r, time.perf_counter())
        return failed

    def fill_asks(self, buf, step: Step, entries: int, rows: int) -> None:
        """What the step's requests ask, into its part of the host buffer."""
        np, at = self.np, 0
        if self.adapter_slots:
            buf[:rows] = -1
            of = [r.adapter for r, toks in step.entries for _ in toks]
            buf[: len(of)] = of
            at = rows
        if not self.own_sampling:
            return
        # a field each; entries that need no token, and places without an entry, are passed over
        ints = buf[at : at + len(self.SAMPLING_INTS) * entries].reshape(-1, entries)
        at += ints.size
        floats = buf[at : at + len(self.SAMPLING_FLOATS) * entries].view(np.float32).reshape(-1, entries)
        at += floats.size
        ids = buf[at : at + self.max_bias * entries].reshape(entries, self.max_bias)
        bias = buf[at + ids.size : at + 2 * ids.size].view(np.float32).reshape(entries, self.max_bias)
        ints[:], floats[:], ids[:] = np.array([[-1], [0], [0], [-1], [0]]), np.array([[1], [0], [0], [0], [1], [0], [0]], np.float32), -1
        plain = Sampling()
        places, own_ints, own_floats = [], [], []
        for e, (r, toks) in enumerate(step.entries):
            if not self.wants_token(r, toks):
                continue
            if not r.output:  # the first token comes next: its history is the prompt
                host = self.torch.tensor(r.prompt_ids, dtype=self.torch.int32).pin_memory()
                self.history[r.history, : len(host)].copy_(host, non_blocking=True)
            s = r.sampling or plain
            mask = step.masks[r.id] if r.id in step.masks else self.mask_of(r)
            places.append(e)
            own_ints.append((r.history, len(r.prompt_ids) + len(r.output), len(r.prompt_ids), mask, s.top_k))
            own_floats.append((s.repetition, s.presence, s.frequency, s.temperature, s.top_p, s.min_p, r.rng.random()))
            if s.bias:
                ids[e, : len(s.bias)] = list(s.bias)
                bias[e, : len(s.bias)] = list(s.bias.values())
        if places:
            ints[:, places], floats[:, places] = np.array(own_ints).T, np.array(own_floats).T

    def asks_views(self, dev, entries: int, rows: int, first: int | None = None, first_rows: int | None = None):
        """The model's view of what was filled in, of the first entries and rows."""
        if not len(dev):
            return {}
        from .models import Asks
        from .ops import Draw, Rules

        asks, at, E = Asks(), 0, entries if first is None else first
        if self.adapter_slots:
            asks.adapters = dev[: rows if first_rows is None else first_rows]
            at = rows
        if self.own_sampling:
            f = {}
            for name in self.SAMPLING_INTS + self.SAMPLING_FLOATS:
                f[name] = dev[at : at + E]
                if name in self.SAMPLING_FLOATS:
                    f[name] = f[name].view(self.torch.float32)
                at += entries
            biases = {}
            if self.max_bias:
                n = self.max_bias
                biases = {"bias_ids": dev[at : at + E * n].view(E, n), "bias": dev[at + entries * n :][: E * n].view(self.torch.float32).view(E, n)}
            asks.draw = Draw(*(f.pop(name) for name in ("temperature", "uniform", "top_k", "top_p", "min_p")))
            asks.rules = Rules(history=self.history, masks=self.masks, **f, **biases)
        return {"asks": asks}

    def decode_layout(self) -> list[int]:
        """ids, cached_lens, num_decoding, block table, state slots of a pure-decode step, and what the requests ask, sized for the largest
        batch; a bucket of b rows uses the first b of each (same start addresses for every bucket)."""
        B = self.max_batch_size
        return [B, B, 1, B * self.max_pages, B, self.asks_size(B, B)]

    def table_row(self, r: Request):
        """The request's block-table row as an int32 array, extended in place as pages are appended."""
        n, row = self.rows.get(r.id, (0, None))
        if row is None:
            row = self.np.zeros(self.max_pages, self.np.int32)
        if n < len(r.pages):
            row[n : len(r.pages)] = r.pages[n:]
            self.rows[r.id] = (len(r.pages), row)
        return row

    def fill_mixed(self, step: Step, n_pad: int, live: int | None = None):
        """Build the step's metadata on the host (scaffold.plan_step = the reference's fill_inputs), one copy."""
        nd, num_entries = step.num_decoding, self.step_entries(n_pad, live)
        plan = self.S.plan_step([r.cached_len for r, _ in step.entries[:nd]],
                           [(r.cached_len, len(t)) for r, t in step.entries[nd:]], n_pad, num_entries, self.block_m)
        sizes = self.mixed_layout(n_pad, live)
        buf = self.np_mixed[: sum(sizes)]
        offs = [0]
        for n in sizes:
            offs.append(offs[-1] + n)
        ids = [tok for _, toks in step.entries for tok in toks]
        buf[offs[0] : offs[0] + len(ids)] = ids
        buf[offs[0] + len(ids) : offs[1]] = 0
        for i, key in enumerate(("positions", "seq_ids", "cu_seqlens", "cached", "cu_cached", "tile_start", "num_decoding"), 1):
            assert len(plan[key]) == sizes[i]
            buf[offs[i] : offs[i + 1]] = plan[key]
        table = buf[offs[8] : offs[9]].reshape(num_entries, self.max_pages)
        for i, (r, _) in enumerate(step.entries):
            table[i] = self.table_row(r)
        table[len(step.entries)] = self.scratch_row  # the padding entry lives on the scratch run
        table[len(step.entries) + 1 :] = 0
        slots = buf[offs[9] : offs[10]]
        slots[:] = -1
        slots[: len(step.entries)] = [r.slot for r, _ in step.entries]
        self.fill_asks(buf[offs[10] : offs[11]], step, num_entries, n_pad)
        self.dev_mixed[: len(buf)].copy_(self.host_mixed[: len(buf)], non_blocking=True)
        return plan["cu_cached"][-1]

    def mixed_views(self, n_pad: int, prefix_tokens: int = 0, live: int | None = None):
        S, sizes = self.S, self.mixed_layout(n_pad, live)
        v = self.dev_mixed[: sum(sizes)].split(sizes)
        inp = S.StepInputs(ids=v[0], positions=v[1], seq_ids=v[2], cu_seqlens=v[3], cached_lens=v[4], cu_cached=v[5],
                           tile_start=v[6], num_decoding=v[7], block_table=v[8].view(-1, self.max_pages),
                           prefix_tokens=prefix_tokens, block_m=self.block_m, slots=v[9])
        if self.prefix is None:
            return inp, None
        # a step whose cached prefixes exceed the scratch gets a one-off buffer
        pk, pv = self.prefix if prefix_tokens <= self.prefix_capacity else self.model.make_prefix(prefix_tokens)
        return inp, S.PrefixScratch(pk, pv, inp.cu_cached)

    def decode_views(self, b: int):
        B = self.max_batch_size
        ids, cached, nd, table, slots, asks = self.dev_decode.split(self.decode_layout())
        return ids[:b], cached[:b], nd, table.view(B, self.max_pages)[:b], slots[:b], self.asks_views(asks, B, B, b, b)

    # ------------------------------------------------------------------ execution
    def forward_mixed(self, n_pad: int, prefix_tokens: int = 0, live: int | None = None):
        inp, prefix = self.mixed_views(n_pad, prefix_tokens, live)
        state = {} if self.slots is None else {"slots": inp.slots}
        sizes = self.mixed_layout(n_pad, live)
        state |= self.asks_views(self.dev_mixed[sum(sizes[:-1]) : sum(sizes)], self.step_entries(n_pad, live), n_pad)
        return self.model.step(self.caches, inp, inp.ids, inp.cached_lens, inp.block_table, inp.num_decoding, prefix, **state)

    def forward_decode(self, b: int):
        ids, cached, nd, table, slots, asks = self.decode_views(b)
        state = ({} if self.slots is None else {"slots": slots}) | asks
        return self.model.step(self.caches, None, ids, cached, table, nd, **state)

    def capture_graph(self, run):
        """Two eager runs first (engine.py:432-449), then the recording; returns (graph, the step's output)."""
        torch = self.torch
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                run()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=self.graph_pool):
            out = run()
        return g, out

    def capture(self) -> None:
        """One graph per batch bucket (rows beyond the step's requests are not decoding: num_decoding is read
        on the device) and one per token bucket (any mix of entries that fits, engine.py:412-430).  The dummy
        inputs during capture are a single padding entry on the scratch run, so what the warm-up writes is
        harmless."""
        self.dev_decode.zero_()  # nothing decodes
        if n := self.decode_layout()[-1]:
            self.fill_asks(self.np_decode[-n:], Step([], 0), self.max_batch_size, self.max_batch_size)
            self.dev_decode[-n:].copy_(self.host_decode[-n:])
        for b in reversed(self.graph_buckets):
            self.decode_graphs[b] = self.capture_graph(lambda b=b: self.forward_decode(b))
        for n in reversed(self.token_buckets):
            self.fill_mixed(Step([], 0), n)
            self.mixed_graphs[n] = self.capture_graph(lambda n=n: self.forward_mixed(n))
        self.torch.cuda.synchronize()
        # the warm-up steps ran on all-idle inputs: a status bit here is a fault of the path, not of the data
        bits = self.K.check_status(self.device)
        if bits:
            raise RuntimeError(f"device status word {bits:#x} set while the step graphs were captured")

    def run(self, step: Step):
        """Execute a planned step; the outputs' first entries / rows are the step's own."""
        if self.adapters is not None and self.model.adapters is not self.adapters:
            raise RuntimeError("the model was given other slots for adapters than the engine was made with")
        return self.run_decode(step) if step.decode_only else self.run_mixed(step)

    def run_decode(self, step: Step):
        torch = self.torch
        t_in = time.perf_counter()
        B = len(step.entries)
        b = next(x for x in self.graph_buckets if x >= B)
        Bm, buf = self.max_batch_size, self.np_decode
        buf[:B] = [t[0] for _, t in step.entries]
        buf[Bm : Bm + B] = [r.cached_len for r, _ in step.entries]
        buf[B:Bm] = 0
        buf[Bm + B : 2 * Bm] = 0
        buf[2 * Bm] = B
        slots_at = 2 * Bm + 1 + Bm * self.max_pages
        table = buf[2 * Bm + 1 : slots_at].reshape(Bm, self.max_pages)
        for i, (r, _) in enumerate(step.entries):
            table[i] = self.table_row(r)
        table[B:] = 0
        buf[slots_at : slots_at + Bm] = -1
        buf[slots_at : slots_at + B] = [r.slot for r, _ in step.entries]
        self.fill_asks(buf[slots_at + Bm :], step, Bm, Bm)
        self.dev_decode.copy_(self.host_decode, non_blocking=True)
        self.seconds["inputs"] += time.perf_counter() - t_in
        if b in self.decode_graphs:
            g, out = self.decode_graphs[b]
            g.replay()
            self.steps_run["decode_graph"] += 1
        else:
            with torch.inference_mode():
                out = self.forward_decode(b)
            self.steps_run["eager"] += 1
        return out

    def run_mixed(self, step: Step):
        torch = self.torch
        N = step.num_tokens
        n_pad = next((x for x in self.token_buckets if x >= N), N)
        live = None if n_pad in self.mixed_graphs else len(step.entries)
        t_in = time.perf_counter()
        prefix_tokens = self.fill_mixed(step, n_pad, live)
        self.seconds["inputs"] += time.perf_counter() - t_in
        if n_pad in self.mixed_graphs and (self.prefix is None or prefix_tokens <= self.prefix_capacity):
            g, out = self.mixed_graphs[n_pad]
            g.replay()
            self.steps_run["mixed_graph"] += 1
        else:
            with torch.inference_mode():
                out = self.forward_mixed(n_pad, prefix_tokens, live)
            self.steps_run["eager"] += 1
        return out
