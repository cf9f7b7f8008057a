"""Generation with drafted tokens: a small model proposes, the served model checks several positions in one step.

A round: the draft model decodes ``drafts`` tokens for every request, one after another, and leaves the distribution of each
(``kernels.token_probabilities``); the target model runs the last token and the drafts as one step with logits at all of them;
``kernels.verify_drafts`` keeps a prefix and draws one more token, distributed as the target model alone would have drawn it (greedy
requests get exactly the target's tokens). What a round leaves on the device (tokens, how many were kept, the requests'
lengths) is what the next one starts from: the block tables of both models follow the lengths there (``kernels.step_tables`` ahead
of a step, ``kernels.trim_tables`` behind the verification), and the host reads a round's tokens while the next one runs.

Every request may run the target with a low-rank adapter of its own (``adapter_slots``); the draft model runs as it is, which
costs accepted drafts, not correctness.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from ..ops import kernels
from ..sampling.params import RandomStream, SamplingParams
from .loading import load_model
from .step import Segment, StepContext, StepEngine


class _Side:
    """One of the two models with pages of its own and block tables that live on the device."""

    def __init__(self, model, page_size: int, requests: int, positions: int, step_tokens: int, logit_rows: int, status: torch.Tensor):
        """``status``: a word for every call of the step tables that a round makes (int32, on the device)."""
        stride = (positions + page_size - 1) // page_size
        pool = requests * stride
        self.model, self.page_size, self.requests = model, page_size, requests
        self.steps = StepEngine(model, page_size=page_size, n_pages=pool, max_requests=requests, max_step_tokens=step_tokens, max_logit_rows=logit_rows)
        cache = self.steps.cache
        if len(cache.groups) != 1 or cache.groups[0].need.window or cache.groups[0].need.chunk or cache.state_layers:
            raise ValueError("drafted tokens: the models' layers must keep the keys and values of every position, and no other state (a refused "
                             "draft is taken back by forgetting its positions)")
        dev = model.device
        self.tables = torch.full((requests, stride), -1, dtype=torch.int32, device=dev)
        self.held = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free = torch.arange(pool, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), pool, dtype=torch.int32, device=dev)
        self.status = status
        self.row_start = torch.empty(requests + 1, dtype=torch.int32, device=dev)
        self.row_req, self.positions, self.slots = (torch.zeros(step_tokens, dtype=torch.int32, device=dev) for _ in range(3))
        # a step's tokens and counts are copied here: recorded launches name where they lie
        self.tokens, self.counts = torch.zeros(step_tokens, dtype=torch.int32, device=dev), torch.zeros(requests, dtype=torch.int32, device=dev)
        self.all_rows = torch.arange(max(step_tokens, logit_rows), dtype=torch.int32, device=dev)
        self.no_slots = torch.zeros(requests, dtype=torch.int32, device=dev)

    def forward(self, tokens: torch.Tensor, counts: Sequence[int], counts_dev: torch.Tensor, lengths: torch.Tensor, bounds: Sequence[int],
                logits: bool, row_adapter: Optional[torch.Tensor] = None, word: int = 0) -> Optional[torch.Tensor]:
        """A step of ``counts`` tokens a request behind the ``lengths`` cached ones (on the device; ``bounds``: what they are at
        most), with logits at every row or none. ``word``: the status word of the call that makes its tables. A refused call leaves the tables of the
        step before, on which the model must not run: so it is refused here already where the bounds leave room for it."""
        T, R = tokens.numel(), self.requests
        pages = [(b + n + self.page_size - 1) // self.page_size for b, n in zip(bounds, counts)]
        if max(pages) > self.tables.shape[1] or sum(pages) > self.free.numel():
            raise RuntimeError(f"step tables: {sum(pages)} pages, up to {max(pages)} a request, of {self.free.numel()} and {self.tables.shape[1]}")
        self.counts.copy_(counts_dev)
        kernels.step_tables(lengths, self.counts, self.tables, self.held, self.free, self.n_free, self.page_size, self.row_start,
                            self.row_req[:T], self.positions[:T], self.slots[:T], self.status[word:word + 1])
        # (behind the tables: a copy waits for all kernels ahead of it, and the model's first kernel for the copy. Its kernels read the tables early.)
        self.tokens[:T].copy_(tokens)
        views = {"tokens": self.tokens[:T], "positions": self.positions[:T], "row_req": self.row_req[:T], "logit_rows": self.all_rows[:T if logits else 0],
                 "state_slots": self.no_slots, "seg_start": self.row_start[:R], "seg_len": self.counts, "tables": [self.tables]}
        if row_adapter is not None:
            views["row_adapter"] = row_adapter
        segments, row = [], 0
        for r, n in enumerate(counts):
            segments.append(Segment(r, row, n, bounds[r], 0, False))
            row += n
        steps = self.steps
        steps._aux_calls = 0
        ctx = StepContext(steps, T, R, T if logits else 0, segments, views)
        with kernels.on_current_stream():
            steps._begin_adapters(ctx)
            return self.model.forward(ctx)

    def begin(self) -> None:
        """Ahead of the steps of a round, or of a portion of prompts: looks at the kernels' status behind those that have finished. ``end``: behind them (once a
        round: the engine remembers a few places only, and waits for the oldest of them)."""
        self.steps._poll_status(wait=False)
        self._failures = kernels.status_failures(self.steps.device)

    def end(self) -> None:
        self.steps._post_status(self._failures)

    def trim(self, lengths: torch.Tensor) -> None:
        kernels.trim_tables(lengths, self.tables, self.held, self.free, self.n_free, self.page_size, self.status[-1:])


class SpeculativeEngine:
    def __init__(self, model_dir: str, draft_dir: str, drafts: int = 4, dtype: str = "bfloat16", device: str = "cuda:0", max_running: int = 8,
                 max_seq_len: int = 2048, page_size: int = 16, step_tokens: int = 2048, decode_weight_copy: bool = True,
                 adapter_slots: int = 0, adapter_rank: int = 16, weights: str = "native"):
        """``model_dir``, ``draft_dir``: the served and the proposing model, of one vocabulary. ``drafts``: tokens proposed a
        round (fewer where a request that runs is nearer to the end of the models' contexts than that). ``max_seq_len``: positions of a request at most, of the
        prompt and all generated tokens but the last, which is not fed. ``weights``: of the served model (the draft's are native). The other arguments are ``Engine``'s."""
        if adapter_slots and weights != "native":
            raise ValueError("drafted tokens: adapters go with native weights")
        if drafts < 1 or max_running < 1:
            raise ValueError("drafted tokens: drafts and max_running must be positive")
        self.drafts, self.requests, self.page_size = drafts, max_running, page_size
        room = max_seq_len + drafts                # (positions that a full round may write behind the last one that stays)
        target = load_model(model_dir, dtype=dtype, device=device, max_position=room, weight_tiles=decode_weight_copy, weights=weights)
        draft = load_model(draft_dir, dtype=dtype, device=device, max_position=room, weight_tiles=decode_weight_copy)
        if target.vocab_size != draft.vocab_size:
            raise ValueError(f"drafted tokens: the models' vocabularies differ ({target.vocab_size} and {draft.vocab_size})")
        self.positions = min(target.max_position, draft.max_position)
        self.context = min(max_seq_len, self.positions)
        if self.context < 1:
            raise ValueError("drafted tokens: the context is too short")
        self.vocab, self.device = target.vocab_size, target.device
        R, K, V = max_running, drafts, target.vocab_size
        self.step_tokens = max(step_tokens, R * (K + 1))
        # how the calls of a round's step tables went (K + 1 steps and the trimming, a row a side)
        self._status = torch.zeros(2, K + 2, dtype=torch.int32, device=target.device)
        self.target = _Side(target, page_size, R, self.positions, self.step_tokens, R * (K + 1), self._status[0])
        self.draft = _Side(draft, page_size, R, self.positions, self.step_tokens, R, self._status[1])
        if adapter_slots:
            self.target.steps.enable_adapters(adapter_slots, adapter_rank)
        dev = self.device
        ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)      # noqa: E731
        self._lengths, self._current, self._ends = ints(R), ints(R), ints(R)
        self._at = ints(K + 1, R)                                   # lengths of the drafting steps
        self._ids, self._drafted, self._fed = ints(K, R), ints(R * K), ints(R * (K + 1))
        self._counts = ints(R)
        # of a round of k drafts: drafts a request, rows a request, its first row
        self._some = [(ints(R) + k, ints(R) + (k + 1), torch.arange(R, dtype=torch.int32, device=dev) * (k + 1)) for k in range(K + 1)]
        # what a round leaves for the host, in one piece (a copy of columns would wait for the device): the tokens, how many drafts were kept, and which calls of
        # the step tables were refused in the batch so far
        self._out = ints((R + 2) * (K + 2))
        self._tokens, self._accepted, self._refused = self._out.split([R * (K + 1), R, 2 * (K + 2)])
        self._refused = self._refused.view(2, K + 2)
        self._probs = torch.empty(K, R, V, dtype=torch.float32, device=dev)
        self._scratch = torch.empty(R, V, dtype=torch.float32, device=dev)
        self._work = torch.empty(R * (K + 1), 4, dtype=torch.float32, device=dev)
        self._temperature = torch.zeros(R, dtype=torch.float32, device=dev)
        self._no_top_k, self._no_top_p = ints(R), torch.ones(R, dtype=torch.float32, device=dev)
        self._adapters, self._row_adapter = ints(R) - 1, ints(self.step_tokens)      # (one place for every step: recorded launches name it)
        # two rounds may be in flight: numbers on their way in, tokens on their way out
        n = R * (2 * K + 1)
        self._numbers_host = [torch.zeros(n).pin_memory() for _ in range(3)]
        self._numbers = [torch.zeros(n, device=dev) for _ in range(3)]
        self._out_host = [torch.zeros(self._out.numel(), dtype=torch.int32).pin_memory() for _ in range(3)]
        self._done = [None] * 3
        self.rounds = self.proposed = self.kept = 0

    def load_adapter(self, slot: int, folder: str) -> None:
        """Reads a low-rank adapter of the target model into a slot (``Engine.load_adapter``)."""
        from ..weights.adapters import read_adapter
        pairs, scale = read_adapter(folder)
        self.target.steps.put_adapter(slot, pairs, scale)

    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 16, temperature=0.0, seed: int = 1,
                 stop_ids: Sequence[int] = (), adapters: Optional[Sequence[int]] = None) -> List[List[int]]:
        """Up to ``max_new_tokens`` for every prompt, ``max_running`` of them at a time; ``temperature``: one number, or one a prompt (0:
        greedy). Request i draws with seed ``seed + i`` and runs the target with the adapter in slot ``adapters[i]`` (-1: none)."""
        temps = list(temperature) if hasattr(temperature, "__len__") else [float(temperature)] * len(prompts)
        slots = list(adapters) if adapters is not None else [-1] * len(prompts)
        if len(temps) != len(prompts) or len(slots) != len(prompts):
            raise ValueError("generate: a temperature and an adapter for every prompt")
        have = self.target.steps.adapter_step.slots if self.target.steps.adapter_step is not None else 0
        for p, t, a in zip(prompts, temps, slots):
            SamplingParams(temperature=float(t))               # (refuses what is no temperature)
            if not 1 <= len(p) or len(p) + max_new_tokens - 1 > self.context:
                raise ValueError(f"generate: a prompt of {len(p)} tokens and {max_new_tokens} more do not fit in {self.context} positions")
            if any(not 0 <= int(x) < self.vocab for x in p):
                raise ValueError("generate: token id out of range")
            if a >= have:
                raise ValueError(f"generate: there is no adapter slot {a}")
        out: List[List[int]] = []
        for at in range(0, len(prompts), self.requests):
            some = slice(at, at + self.requests)
            out += self._batch([list(p) for p in prompts[some]], max_new_tokens, temps[some], [seed + at + i for i in range(len(prompts[some]))],
                               set(stop_ids), slots[some])
        return out

    # ------------------------------------------------------------------ one batch
    def _batch(self, prompts, max_new, temps, seeds, stop_ids, slots) -> List[List[int]]:
        R, n, dev = self.requests, len(prompts), self.device
        if max_new <= 0:
            return [[] for _ in prompts]
        fill = lambda t, values, rest: t.copy_(torch.tensor(list(values) + [rest] * (R - n), dtype=t.dtype))      # noqa: E731
        self._lengths.zero_()
        self._refused.zero_()
        self._status.zero_()
        for side in (self.target, self.draft):
            side.trim(self._lengths)                           # (whatever an earlier batch held)
        self._refused |= self._status
        fill(self._temperature, temps, 0.0)
        fill(self._adapters, slots, -1)
        fill(self._current, [p[-1] for p in prompts], 0)
        # places without a request, and those whose request has ended (0 as well), run along from position 0 on
        ends = [len(p) - 1 + max_new for p in prompts] + [0] * (R - n)
        self._ends.copy_(torch.tensor(ends, dtype=torch.int32))
        adapted = any(a >= 0 for a in slots)
        self._prefill(prompts, adapted)
        streams = [RandomStream(s) for s in seeds]
        lengths = [len(p) - 1 for p in prompts] + [0] * (R - n)          # as of the rounds that have been collected
        results: List[List[int]] = [[] for _ in prompts]
        alive = [True] * n
        pending, ahead = None, 0                               # the round that is not collected yet, and the tokens that it may give
        rounds = 0
        while True:
            now = None
            if any(alive) and rounds < max_new:                # (a round gives every request a token at least)
                bounds = [min(l + ahead, e - 1) if e else 0 for l, e in zip(lengths, ends)]
                drafts = min(self.drafts, self.positions - 1 - max(bounds))          # (a round of k drafts writes k positions behind the length)
                now = self._round(rounds % 3, drafts, streams, temps, bounds, adapted)
                rounds += 1
            if pending is not None:
                self._collect(pending, lengths, ends, results, alive, max_new, stop_ids)
            if now is None:
                break
            pending, ahead = now, drafts + 1
        for side in (self.target, self.draft):
            side.steps.check_status()
        return results

    def _prefill(self, prompts, adapted: bool) -> None:
        """All of every prompt but its last token, in portions of the step's token limit."""
        R, dev = self.requests, self.device
        fed = [0] * R
        total = [len(p) - 1 for p in prompts] + [0] * (R - len(prompts))
        while any(f < t for f, t in zip(fed, total)):
            budget, counts, tokens, rows = self.step_tokens, [], [], []
            for r in range(R):
                take = min(total[r] - fed[r], budget)
                budget -= take
                counts.append(take)
                if take:
                    tokens += prompts[r][fed[r]:fed[r] + take]
                    rows += [r] * take
            ids = torch.tensor(tokens, dtype=torch.int32).to(dev)
            self._counts.copy_(torch.tensor(counts, dtype=torch.int32))
            row_adapter = None
            if adapted:
                row_adapter = self._row_adapter[:len(rows)]
                row_adapter.copy_(self._adapters[torch.tensor(rows).to(dev)])
            for side, adapter in ((self.target, row_adapter), (self.draft, None)):
                side.begin()
                side.forward(ids, counts, self._counts, self._lengths, fed, False, adapter)
                side.end()
            self._refused |= self._status
            self._lengths += self._counts
            fed = [f + c for f, c in zip(fed, counts)]

    def _round(self, turn: int, K: int, streams, temps, bounds, adapted: bool):
        """Launches a round of ``K`` drafts; its tokens are on their way to the host behind the returned event."""
        R = self.requests
        if self._done[turn] is not None:
            self._done[turn].synchronize()
        host, numbers = self._numbers_host[turn], self._numbers[turn]
        for r, stream in enumerate(streams):
            if temps[r] > 0:
                for j in range(K):
                    host[j * R + r] = stream.next_uniform()                      # the draft's draw
                for j in range(K):
                    host[K * R + r * K + j] = stream.next_uniform()              # whether it is kept
                host[2 * K * R + r] = stream.next_uniform()                      # the token behind the kept ones
        numbers.copy_(host, non_blocking=True)
        accept, draw = numbers[K * R:2 * K * R].view(R, K), numbers[2 * K * R:2 * K * R + R]
        drafts, rows, starts = self._some[K]
        drafted, fed, result = self._drafted[:R * K].view(R, K), self._fed[:R * (K + 1)].view(R, K + 1), self._tokens[:R * (K + 1)].view(R, K + 1)
        # the drafts, and one step more that only leaves the last one's keys and values
        torch.add(self._lengths, torch.arange(K + 1, dtype=torch.int32, device=self.device)[:, None], out=self._at[:K + 1])
        ones = [1] * R
        self.draft.begin()
        for j in range(K + 1):
            tokens = self._current if j == 0 else self._ids[j - 1]
            logits = self.draft.forward(tokens, ones, self._some[0][1], self._at[j], [b + j for b in bounds], j < K, word=j)
            if j < K:
                kernels.token_probabilities(logits, self._temperature, self._probs[j])
                kernels.argmax(logits, self._ids[j])
                kernels.sample(logits, self._scratch, self._temperature, self._no_top_k, self._no_top_p, numbers[j * R:(j + 1) * R], self._ids[j])
        self.draft.end()
        drafted.copy_(self._ids[:K].t())
        fed[:, 0].copy_(self._current)
        fed[:, 1:].copy_(drafted)
        row_adapter = None
        if adapted:
            row_adapter = self._row_adapter[:R * (K + 1)]
            row_adapter.view(R, K + 1).copy_(self._adapters[:, None].expand(R, K + 1))
        self.target.begin()
        logits = self.target.forward(fed.view(-1), [K + 1] * R, rows, self._lengths, bounds, True, row_adapter)
        self.target.end()
        kernels.verify_drafts(logits, starts, drafted, drafts, self._probs[:K].transpose(0, 1), self._temperature, accept, draw, result, self._accepted, self._work)
        # the next round starts behind what was kept; requests that have ended from nothing
        self._current.copy_(result.gather(1, self._accepted.long()[:, None])[:, 0])
        self._lengths += self._accepted + 1
        ended = self._lengths >= self._ends
        self._lengths.masked_fill_(ended, 0)
        self._ends.masked_fill_(ended, 0)
        for side in (self.target, self.draft):
            side.trim(self._lengths)
        self._refused |= self._status
        self._out_host[turn].copy_(self._out, non_blocking=True)
        event = torch.cuda.Event()
        event.record()
        self._done[turn] = event
        return turn, K, event

    def _collect(self, pending, lengths, ends, results, alive, max_new: int, stop_ids) -> None:
        """A round's tokens into ``results``; ``lengths`` and ``ends`` follow those on the device."""
        turn, K, event = pending
        event.synchronize()
        R = self.requests
        out = self._out_host[turn].tolist()
        kept, statuses = out[R * (self.drafts + 1):R * (self.drafts + 2)], out[R * (self.drafts + 2):]
        refused = next((status for status in statuses if status), 0)
        if refused:
            raise RuntimeError(f"step tables were refused (status {refused})")
        self.rounds += 1
        for r in range(R):
            lengths[r] += kept[r] + 1
            if lengths[r] >= ends[r]:
                lengths[r] = ends[r] = 0
        for r, result in enumerate(results):
            if not alive[r]:
                continue
            self.proposed += K
            self.kept += kept[r]
            for token in out[r * (K + 1):r * (K + 1) + kept[r] + 1]:
                result.append(int(token))
                if token in stop_ids or len(result) == max_new:
                    alive[r] = False
                    break
