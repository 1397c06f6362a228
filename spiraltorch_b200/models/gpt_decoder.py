"""Answering token by token with a :class:`~spiraltorch_b200.models.gpt.GPTModel`: keys and values in an 8-bit paged cache.

Every call is one pass of the model over the new tokens of all sequences, one after another in the rows of one matrix:
:func:`ops.paged.plan` takes pages and maps the rows, then per layer the fused projection, rotary positions, :func:`ops.paged.store` and
attention over the cache.  Where all that is added is whole prompts of ``DENSE_FROM`` tokens and more, they read the cache back instead
(:func:`ops.paged.read`) and run ``ops.attention`` over it, which knows that a causal prompt's first tokens see few keys; so a prompt sees the same keys and
values that later tokens do, by weights that are rounded to bf16 there and to fp16 otherwise.

A part of a prompt beside single tokens of other sequences slows these: attention takes its tile from the longest part (``max_queries``).  63 single tokens at
4096 with 16 heads take 170 us, with a part of 256 tokens in the same call 497, where the part alone takes 39.

A step of few sequences is little but reading weights: ``weight_bits=4`` (and ``head_bits=4`` for the logits' product) keeps a copy of the matrices in four bits
(:mod:`ops.int4`), which :meth:`GPTDecoder.refresh` makes anew after an update of the model.

The reference has no counterpart (its language models do not decode with a cache)."""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from ..ops import attention as attn_ops
from ..ops import elementwise as ew
from ..ops import gemm as gemm_ops
from ..ops import int4
from ..ops import native
from ..ops import paged
from ..ops import rotary as rotary_ops
from ..ops import scoring

# Tokens of a whole prompt.  16 heads of 128, us over the cache and read back, one prompt: 512 tokens 22 and 66, 1024 28 and 50, 1536 45 and 51, 2048 71 and 51,
# 4096 167 and 88.  Reading back takes two launches for each prompt, the cache's kernel one for all: four prompts of 2048 188 and 211, of 4096 521 and 353.
DENSE_FROM = 2048


class GeneratedScores(NamedTuple):
    """For every new token of a sequence: its log probability, the entropy of the distribution behind it, the likeliest tokens and theirs."""
    logprob: list
    entropy: list
    top_ids: list
    top_logprobs: list


class GPTDecoder:
    """``sequences`` places for sequences of up to ``max_length`` tokens over ``pages`` pages (default: enough for all of them).

    The lengths are kept on the host as well (``held``), so that a call that does not fit is refused before anything is launched.  Replays of a captured
    :meth:`step` do not pass through them: once a step has been captured, every other call first takes them from the device (:meth:`sync`).

    A kernel that gives up (a page that is none, a wait that runs out) leaves an error record; :meth:`extend` and :meth:`step` raise what calls and replays before
    them left, :meth:`generate` what its own passes leave.

    ``weight_bits`` 4: the layers' matrices in four bits, with a scale for every ``group`` inputs; ``head_bits`` 4: those of the logits too."""

    def __init__(self, model, sequences: int, max_length: int, *, pages: Optional[int] = None, page_size: int = 64, weight_bits: int = 16, head_bits: int = 16,
                 group: int = 64):
        cfg = model.cfg
        if model.tp.world != 1:
            raise ValueError("GPTDecoder: tensor-parallel models are not supported")
        if sequences < 1 or max_length < 1:
            raise ValueError(f"GPTDecoder: {sequences} sequences of up to {max_length} tokens")
        if cfg.positional == "learned" and max_length > cfg.seq_len:
            raise ValueError(f"GPTDecoder: learned positions end at {cfg.seq_len}, not at {max_length}")
        if weight_bits not in (4, 16) or head_bits not in (4, 16):
            raise ValueError(f"GPTDecoder: weights of 4 or 16 bits, got {weight_bits} and {head_bits} for the logits")
        if (weight_bits == 4 or head_bits == 4) and model.flat_w.is_cuda and model.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"GPTDecoder: weights of 4 bits are multiplied by bf16 and fp16 activations, not by {model.dtype}")
        self.model, self.sequences, self.max_length, self.page_size = model, sequences, max_length, page_size
        dev = model.flat_w.device
        width = -(-max_length // page_size)
        self.pages = sequences * width if pages is None else pages
        self.cache = [paged.Pages.allocate(self.pages, cfg.n_heads, page_size, cfg.head_dim, dev) for _ in range(cfg.n_layers)]
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((sequences, width), -1, **i32)
        self.free = torch.arange(self.pages, **i32)
        self.free_count = torch.full((1,), self.pages, **i32)
        self.lengths = torch.zeros(sequences, **i32)
        self.held = [0] * sequences
        self._left = self.pages
        self._lost = [False] * sequences        # replays found no page for some of its tokens
        self._waiting = [False] * sequences     # released, and not extended since: steps pass it over
        # the same on the device, for steps: tokens that each place adds; the place of each row and the row of each place, -1 for those that wait
        self._taking = torch.ones(sequences, **i32)
        self._place_of_row, self._row_of_place = torch.arange(sequences, device=dev), torch.arange(sequences, device=dev)
        self._captured = False
        names = [f"h{l}.{n}.weight" for l in range(cfg.n_layers) for n in ("qkv", "proj", "fc1", "fc2")] if weight_bits == 4 else []
        self.weights = {n: int4.quantize(model.p[n], group) for n in names + (["embed.weight"] if head_bits == 4 else [])}

    def refresh(self) -> None:
        """The weights in four bits from what the model's are now, in the memory that captured steps read."""
        for n, held in self.weights.items():
            int4.quantize(self.model.p[n], held.group, out=held)

    def _product(self, x: torch.Tensor, name: str, act: Optional[str] = None) -> torch.Tensor:
        held = self.weights.get(name)
        return gemm_ops.gemm(x, self.model.p[name], act=act) if held is None else int4.linear(x, held, act=act)

    # ---- host side ------------------------------------------------------------------------------------------------------------
    def _blocks(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    @property
    def pages_left(self) -> int:
        self._settle()
        return self._left

    def sync(self) -> None:
        """Takes ``held`` and the free pages from the device, which replays have moved on (waits for it)."""
        block = torch.arange(self.table.shape[1], dtype=torch.int32, device=self.table.device)
        lost = ((self.table < 0) & (block < ((self.lengths + (self.page_size - 1)) // self.page_size)[:, None])).any(1)
        state = torch.cat([self.lengths, lost.int(), self.free_count]).tolist()
        n = self.sequences
        self.held, self._lost, self._left = state[:n], [x > 0 for x in state[n:2 * n]], max(state[-1], 0)

    def _capturing(self) -> bool:
        return self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()

    def _settle(self) -> None:
        if self._captured and not self._capturing():
            self.sync()

    def _need(self, added: Sequence[int]) -> int:
        return sum(self._blocks(h + n) - self._blocks(h) for h, n in zip(self.held, added))

    def _admit(self, added: Sequence[int]) -> None:
        """Refuses what does not fit."""
        for b, (h, n) in enumerate(zip(self.held, added)):
            if n and self._lost[b]:
                raise ValueError(f"GPTDecoder: place {b} lost tokens to replays that found no page; it must be released")
            if h + n > self.max_length:
                raise ValueError(f"GPTDecoder: sequence {b} would have {h + n} tokens, at most {self.max_length}")
        if (need := self._need(added)) > self._left:
            raise ValueError(f"GPTDecoder: {need} pages are needed and {self._left} are left")

    def _commit(self, added: Sequence[int]) -> None:
        self._left -= self._need(added)
        self.held = [h + n for h, n in zip(self.held, added)]

    def _wait(self, waiting: list) -> None:
        if waiting != self._waiting:
            take = ~torch.tensor(waiting)
            self._taking.copy_(take)
            self._row_of_place.copy_(torch.where(take, take.cumsum(0) - 1, -1))
            self._place_of_row.copy_(torch.cat([take.nonzero()[:, 0], torch.full((sum(waiting),), -1)]))
            self._waiting = waiting

    # ---- device side ----------------------------------------------------------------------------------------------------------
    def _pass(self, tokens: torch.Tensor, added: torch.Tensor, last: Optional[torch.Tensor], counts: Sequence[int], by_place: bool = False) -> torch.Tensor:
        """Logits of the rows ``last`` (None: all) of ``tokens`` ``[rows]``, of which sequence ``b`` has ``counts[b]``.  ``by_place``: a token
        and logits for every place; those that wait have rows behind the last sequence, and logits of 0."""
        m, cfg = self.model, self.model.cfg
        H, D, rows, most = cfg.n_heads, cfg.head_dim, tokens.shape[0], max(counts)
        dense = last is not None and all(n == 0 or DENSE_FROM <= n and held == 0 for n, held in zip(counts, self.held))      # as many queries as keys
        step = paged.plan(self.lengths, added, self.table, self.free, self.free_count, page_size=self.page_size, rows=rows)
        resid, x = ew.embedding_forward(tokens, m.p["embed.weight"]), None
        if by_place:      # rows in the order of the plan; a lookup of -1 gives zeros
            resid = ew.embedding_forward(self._place_of_row, resid)
        if cfg.positional == "learned":
            resid = resid + m.p["pos.weight"][step.positions.long().clamp_(max=cfg.seq_len - 1)]      # replays may go on behind the end
        for l in range(cfg.n_layers):
            y, h, _, _ = m._norm_fwd(resid if x is None else x, f"h{l}.norm1", residual=None if x is None else resid)
            if x is not None:
                resid = h
            qkv = self._product(y, f"h{l}.qkv.weight").view(rows, 3, H, D)
            q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
            if m.rope_freq is not None:
                rotary_ops.rotary_(q, k, step.positions, m.rope_freq, interleaved=cfg.rope_interleaved)
            paged.store(k, v, self.cache[l], step.slots)
            o = self._dense(q, l, counts, step.lengths) if dense else paged.attention(q, self.cache[l], self.table, step.starts, step.lengths, max_queries=most)
            a = self._product(o.view(rows, H * D), f"h{l}.proj.weight")
            y, resid, _, _ = m._norm_fwd(a, f"h{l}.norm2", residual=resid)
            u = self._product(y, f"h{l}.fc1.weight", "gelu")
            x = self._product(u, f"h{l}.fc2.weight")
        if last is not None:
            x, resid = x.index_select(0, last), resid.index_select(0, last)
        y, _, _, _ = m._norm_fwd(x, "norm_f", residual=resid)
        if by_place:
            y = ew.embedding_forward(self._row_of_place, y)
        logits = self._product(y, "embed.weight")
        # only now does the step take effect: a call that failed before appended nothing, and what it wrote to the table and the pages is written anew
        self.lengths.copy_(step.lengths)
        self.free_count.copy_(step.free_count)
        return logits

    def _dense(self, q: torch.Tensor, l: int, counts: Sequence[int], lengths: torch.Tensor) -> torch.Tensor:
        o, r = torch.empty(q.shape, dtype=q.dtype, device=q.device), 0
        for b, n in enumerate(counts):
            if n:
                k, v = paged.read(self.cache[l], self.table[b:b + 1], lengths[b:b + 1], n,
                                  torch.bfloat16 if q.is_cuda else torch.float32)
                o[r:r + n] = attn_ops.attention_forward(q[None, r:r + n], k, v, True)[0][0]
                r += n
        return o

    @torch.no_grad()
    def extend(self, tokens: Sequence) -> torch.Tensor:
        """``tokens``: for every sequence the ids to append (a list or a 1-D host tensor; empty: the sequence waits).  Returns the logits behind the last
        token of each sequence that got some, ``[such sequences, vocab]``."""
        if len(tokens) != self.sequences:
            raise ValueError(f"GPTDecoder: tokens for {len(tokens)} of {self.sequences} sequences")
        ids = [torch.as_tensor(t, dtype=torch.int64).reshape(-1) for t in tokens]
        counts = [t.numel() for t in ids]
        flat = torch.cat(ids)
        vocab = self.model.cfg.vocab_size
        if flat.numel() and (int(flat.min()) < 0 or int(flat.max()) >= vocab):
            raise ValueError(f"GPTDecoder: a token id is outside the vocabulary of {vocab}")
        if not flat.numel():
            raise ValueError("GPTDecoder: no tokens")
        if self._capturing():
            raise ValueError("GPTDecoder: extend takes tokens from the host and cannot be captured; step can")
        self._settle()
        native.poll()
        self._admit(counts)
        dev = self.lengths.device
        last = torch.tensor([sum(counts[:b + 1]) - 1 for b, n in enumerate(counts) if n])
        logits = self._pass(flat.to(dev), torch.tensor(counts, dtype=torch.int32, device=dev), last.to(dev), counts)
        self._commit(counts)
        self._wait([w and not n for w, n in zip(self._waiting, counts)])
        return logits

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token for every place: ``tokens`` int64 ``[sequences]`` on the model's device, ids inside the vocabulary (not looked at).
        Returns the logits behind them.  A place that was released waits until :meth:`extend` gives it a new sequence: it takes neither its token nor a
        page, and its logits are 0.

        The call looks at nothing on the device, so it can be captured into a CUDA graph (which appends nothing by itself).  Replays
        follow what :meth:`extend` and :meth:`release` do between them, but no host stands before them: what they append behind a place's last page, or
        when no page is left, is not stored.  Other calls refuse such a place until it is released."""
        if tokens.shape != (self.sequences,) or tokens.dtype != torch.int64 or tokens.device != self.lengths.device:
            raise ValueError(f"GPTDecoder: step takes int64 [{self.sequences}] on {self.lengths.device}, got {tokens.dtype} {tuple(tokens.shape)} on {tokens.device}")
        if self._capturing():
            self._captured = True
            return self._pass(tokens, self._taking, None, [1] * self.sequences, True)
        self._settle()
        native.poll()
        counts = [int(not w) for w in self._waiting]
        if not any(counts):
            raise ValueError("GPTDecoder: every place was released; extend begins a sequence")
        self._admit(counts)
        logits = self._pass(tokens, self._taking, None, counts, any(self._waiting))
        self._commit(counts)
        return logits

    def release(self, which: Sequence[int]) -> None:
        """Ends the sequences of these places and frees their pages; the places wait until :meth:`extend` gives them new ones."""
        if self._capturing():
            raise ValueError("GPTDecoder: release takes places from the host and cannot be captured")
        done = [False] * self.sequences
        for b in which:
            if not 0 <= b < self.sequences:
                raise ValueError(f"GPTDecoder: no place {b}")
            done[b] = True
        paged.release(self.lengths, torch.tensor(done, device=self.lengths.device), self.table, self.free, self.free_count, page_size=self.page_size)
        self._left += sum(self._blocks(h) for h, d in zip(self.held, done) if d)
        self.held = [0 if d else h for h, d in zip(self.held, done)]
        self._lost = [x and not d for x, d in zip(self._lost, done)]
        self._wait([w or d for w, d in zip(self._waiting, done)])

    def generate(self, prompts: Sequence, max_new_tokens: int, *, stop: Optional[int] = None, scores: Optional[int] = None):
        """The likeliest continuation of a prompt in every place, up to ``max_new_tokens`` or the token ``stop`` (which is not returned).
        A place that met ``stop`` waits.  Starts from empty places.

        ``scores``: returns ``(tokens, scores)``, with a :class:`GeneratedScores` of each sequence's tokens and as many of their likeliest alternatives (0 to 32)."""
        self._settle()
        if any(self.held):
            raise ValueError("GPTDecoder: generate starts from empty places; release them first")
        if max_new_tokens < 0 or any(len(p) == 0 for p in prompts):
            raise ValueError("GPTDecoder: prompts need a token at least")
        if scores is not None and not 0 <= scores <= min(scoring.MOST_TOP, self.model.cfg.vocab_size):
            raise ValueError(f"GPTDecoder: scores with 0 to {min(scoring.MOST_TOP, self.model.cfg.vocab_size)} alternatives, got {scores}")
        out, judged = [[] for _ in prompts], [GeneratedScores([], [], [], []) for _ in prompts]
        if max_new_tokens == 0:
            return out if scores is None else (out, judged)
        active = list(range(self.sequences))
        logits = self.extend(prompts)
        while True:
            best = logits.argmax(-1)
            given = None if scores is None else [t.tolist() for t in scoring.token_scores(logits, best, top=scores)]
            going, feed, chosen = [], [[] for _ in prompts], best.tolist()
            native.poll()      # the pass is done
            for i, (b, t) in enumerate(zip(active, chosen)):
                if t != stop:
                    out[b].append(t)
                    if given is not None:
                        for to, values in zip(judged[b], given):
                            to.append(values[i])
                    if len(out[b]) < max_new_tokens:
                        going.append(b)
                        feed[b] = [t]
            if not going:
                return out if scores is None else (out, judged)
            active = going
            logits = self.step(best) if len(going) == self.sequences else self.extend(feed)
