"""Greedy decoding of sequences that come and go, out of a pool of KV pages, on the Qwen3 int8 kernels. No counterpart in the
reference, whose caches are a fixed capacity for every row; a request's contract is its RaggedGraphDecoder's
(research/phase5/ragged.py).

A pool of pages of `page_size` rows is shared by up to 16 sequences (bf16 or int8, per layer and kv head); each holds the
pages that its tokens fill, named by its row of an int32 table, and gives them back when it leaves. A step writes the
batch's rows to their pages (kv_append_paged: q/k norm and rotation on the way, in fp32 and rounded once) and attends over them
(attn_decode_paged). Prompts run through the projections together, behind nothing or behind what a sequence holds already
(a conversation's next turn), and attend to their rows as the cache holds them (kv_read_paged). With top_logprobs the
log probability of every answered token, the distribution's entropy and its most likely tokens come with it
(token_logprobs); score() gives them for a prompt's own tokens.
"""
import contextlib

import torch

from . import ops
from .prefill import _attend, _proj
from .ragged import RaggedEngine, RaggedGraphDecoder, check_ragged


class PagePool:
    """The numbers of the free pages of a pool."""

    def __init__(self, pages):
        if pages < 1:
            raise ValueError('pages must be >= 1')
        self.pages = pages
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free(self):
        return len(self._free)

    def take(self, count):
        if count > len(self._free):
            raise RuntimeError(f'{count} pages asked for, {len(self._free)} of {self.pages} free')
        return [self._free.pop() for _ in range(count)]

    def give(self, pages):
        self._free.extend(reversed(pages))


class PagedEngine(RaggedEngine):
    """RaggedEngine on a pool of pages: add(ids) -> row, any number of step(), extend(row, ids), release(row). After each,
    tokens[row] is the row's newest token (generated, its key not cached yet); with top_logprobs (0 to 32) logprob[row],
    entropy[row], top_ids[row] and top_logprob[row] are of the distribution that it was taken from. capacity: tokens of a
    sequence at most. page_size: int8 pages of 32 rows and more are read faster than smaller ones."""

    def __init__(self, model, batch, pages, capacity, page_size=16, kv_dtype=torch.bfloat16, top_logprobs=None):
        if capacity < 1 or page_size < 1 or page_size & (page_size - 1) or page_size > 1024:
            raise ValueError('capacity must be >= 1 and page_size a power of two up to 1024')
        if top_logprobs is not None and not 0 <= top_logprobs <= 32:
            raise ValueError('top_logprobs must be None or in [0, 32]')
        self.pool, self.page_size, self.top = PagePool(pages), page_size, top_logprobs
        self.columns = -(-capacity // page_size)
        super().__init__(model, batch, capacity, kv_dtype=kv_dtype)
        self.positions.fill_(-1)
        self.idle = torch.ones(batch, dtype=torch.bool, device=self.device)
        self.held = [[] for _ in range(batch)]  # every row's pages
        self.lengths = [0] * batch              # and cached tokens; a row without pages is free
        if self.top is not None:
            self.logprob = torch.zeros(batch, device=self.device)
            self.entropy = torch.zeros(batch, device=self.device)
            self.top_ids = torch.zeros(batch, self.top, dtype=torch.int64, device=self.device)
            self.top_logprob = torch.zeros(batch, self.top, device=self.device)
            self.lp_ws = ops.token_logprobs_ws(batch, self.base.vocab, self.device)

    def _alloc_kv(self):
        b = self.base
        b.kv = None  # the base engine's one-sequence cache is not used here
        self.kv = [ops.kv_pages(self.pool.pages, b.nkv, self.page_size, b.d, b.device,
                                torch.int8 if self.q8 else torch.bfloat16) for _ in range(b.n_layers)]
        self.table = torch.full((self.batch, self.columns), -1, dtype=torch.int32, device=b.device)
        self.q8_ws = ops.attn_paged_ws(self.batch, b.nq, b.nkv, b.d, b.device)

    # ---- rows and their pages
    def _check_row(self, row):
        if not 0 <= row < self.batch:
            raise ValueError(f'row {row} of a batch of {self.batch}')

    def _check_sequence(self, row):
        self._check_row(row)
        if not self.held[row]:
            raise ValueError(f'row {row} has no sequence')

    def reserve(self, row, length):
        """Pages for the first `length` tokens of the row's sequence; all of them or, where the pool has too few, none."""
        self._check_sequence(row)  # (a row that holds pages is taken for one with a sequence)
        self._reserve(row, length)

    def _reserve(self, row, length):
        if length > self.cap:
            raise ValueError(f'{length} tokens exceed the capacity {self.cap}')
        have = len(self.held[row])
        need = -(-length // self.page_size)
        if need > have:
            self.held[row] += self.pool.take(need - have)
            self.table[row, have:need] = torch.tensor(self.held[row][have:], dtype=torch.int32).to(self.device)

    def release(self, row):
        """The row's sequence leaves: its pages are free again, the row idle."""
        self._check_row(row)
        self.table[row] = -1
        self.positions[row] = -1
        self.idle[row] = True
        self._give_back(row, 0, 0)

    def _give_back(self, row, have, length):
        """The row keeps its first `have` pages and `length` tokens."""
        pages = self.held[row][have:]
        self.held[row], self.lengths[row] = self.held[row][:have], length
        self.pool.give(pages)  # (last: an interrupt may lose pages here, but none is ever free and held)

    def reset(self):
        for row in range(self.batch):
            if self.held[row]:
                self.release(row)

    @contextlib.contextmanager
    def _all_or_nothing(self):
        """A change of the batch, whole or, whatever ends it (too few pages, too little memory, an interrupt), not at all: every
        row's pages, length, newest token and its log probabilities are as they were. (What it cached lies behind the lengths.)"""
        before = [(len(pages), length) for pages, length in zip(self.held, self.lengths)]
        state = [self.tokens, self.positions, self.idle]
        if self.top is not None:
            state += [self.logprob, self.entropy, self.top_ids, self.top_logprob]
        saved = [t.clone() for t in state]
        try:
            yield
        except BaseException:
            for r, (have, length) in enumerate(before):
                self.table[r, have:] = -1
                self._give_back(r, have, length)
            for t, old in zip(state, saved):
                t.copy_(old)
            raise

    # ---- prompts
    def _run(self, rows, parts):
        """The ids `parts` (int64 on the device, one tensor a row) behind what the rows hold; -> hidden states of all of them."""
        b = self.base
        counts = [p.numel() for p in parts]
        before = [self.lengths[r] for r in rows]
        for r, f, n in zip(rows, before, counts):
            self._reserve(r, f + n)
        index = torch.tensor(rows, device=self.device)
        table = self.table[index]
        position = torch.tensor(before, device=self.device)
        ends = torch.tensor([0] + counts, device=self.device).cumsum(0)
        longest = max(f + n for f, n in zip(before, counts))
        buf = torch.empty(2, b.nkv, longest, b.d, dtype=torch.bfloat16, device=self.device)

        def attend(i, lay, qkv):
            q, k, v = self._split(qkv)
            q = ops.kv_append_paged(k, v, self.kv[i], table, position, starts=ends, q=q, **self._prologue(lay))
            out, start = [], 0
            for j, (f, n) in enumerate(zip(before, counts)):
                ops.kv_read_paged(self.kv[i], table[j:j + 1], 0, f + n, out=(buf[0, :, :f + n], buf[1, :, :f + n]))
                out.append(_attend(q[start:start + n], buf[0], buf[1], f, b.nq, b.nkv, b.d))
                start += n
            return torch.cat(out)

        h = self._layers(torch.cat(parts), attend)
        for r, f, n in zip(rows, before, counts):
            self.lengths[r] = f + n
        return h, index, ends[1:] - 1

    def _answer(self, logits, tokens, index=None):
        """The log probabilities of `tokens` under `logits`, of all rows or of rows `index`."""
        if self.top is None:
            return
        if index is None:
            ops.token_logprobs(logits, tokens, top=self.top, ws=self.lp_ws,
                               out=(self.logprob, self.entropy) + ((self.top_ids, self.top_logprob) if self.top else (None, None)))
            return
        found = ops.token_logprobs(logits, tokens, top=self.top)
        for mine, t in zip((self.logprob, self.entropy, self.top_ids, self.top_logprob), found):
            if t is not None:
                mine[index] = t

    def _prefill_rows(self, rows, parts):
        b = self.base
        with self._all_or_nothing():
            h, index, last = self._run(rows, parts)
            logits = _proj(ops.rmsnorm(h[last], b.final_norm, b.eps), b.w_lm, b.s_lm)
            tokens = ops.argmax_rows(logits)
            self._answer(logits, tokens, index)
            self.tokens[index] = tokens
            self.positions[index] = torch.tensor([self.lengths[r] for r in rows], device=self.device)
            self.idle[index] = False

    def _ids(self, ids):
        ids = ids.reshape(-1).to(device=self.device, dtype=torch.int64)
        if ids.numel() < 1:
            raise ValueError('a prompt has at least one token')
        return ids

    @torch.no_grad()
    def add(self, ids):
        """A new sequence with the prompt `ids` (int64 [p]) -> its row."""
        return self.add_all([ids])[0]

    @torch.no_grad()
    def add_all(self, prompts):
        """Several new sequences, whose prompts run together -> their rows."""
        if not prompts:
            return []
        rows = [r for r in range(self.batch) if not self.held[r]][:len(prompts)]
        if len(rows) < len(prompts):
            raise RuntimeError(f'{len(prompts)} sequences for {len(rows)} free rows')
        self._prefill_rows(rows, [self._ids(p) for p in prompts])
        return rows

    @torch.no_grad()
    def extend(self, row, ids):
        """The sequence goes on with `ids` behind its newest token (which is run with them)."""
        self._check_sequence(row)
        self._prefill_rows([row], [torch.cat([self.tokens[row:row + 1], self._ids(ids)])])

    def _check_anew(self, lengths, counts, free):
        """Whether sequences with prompts of `lengths` tokens, that grow to counts tokens, have room in `free` pages."""
        for n, count in zip(lengths, counts):
            if n < 1 or count > self.cap:
                raise ValueError(f'a prompt of {n} tokens, a sequence of {count}: at least one, and the capacity is {self.cap}')
        need = sum(-(-n // self.page_size) for n in counts)
        if need > free:
            raise RuntimeError(f'{need} pages asked for, {free} of {self.pool.pages} free once the rows have left')

    @torch.no_grad()
    def prefill(self, prompts, lengths):
        """All rows anew: right-padded prompts [batch, Pmax] and their lengths. The sequences that there are leave once
        the prompts are found to fit."""
        if prompts.dim() != 2 or len(prompts) != self.batch or len(lengths) != self.batch:
            raise ValueError('prefill takes a prompt and its length for every row')
        lengths = [int(n) for n in lengths]
        if max(lengths) > prompts.shape[1]:
            raise ValueError(f'a length of {max(lengths)} of prompts [{self.batch}, {prompts.shape[1]}]')
        self._check_anew(lengths, lengths, self.pool.pages)
        parts = [self._ids(prompts[r, :n]) for r, n in enumerate(lengths)]
        self.reset()
        self._prefill_rows(list(range(self.batch)), parts)

    @torch.no_grad()
    def prefill_row(self, row, ids):
        """One row anew with the prompt `ids` (int64 [p]). A sequence that it has leaves once the prompt is found to fit."""
        self._check_row(row)
        ids = self._ids(ids)
        self._check_anew([ids.numel()], [ids.numel()], self.pool.free + len(self.held[row]))
        self.release(row)
        self._prefill_rows([row], [ids])

    @torch.no_grad()
    def score(self, ids, top=0, rows_at_once=512):
        """What the model gives a text: (logprob, entropy, top_ids, top_logprobs) of its tokens 1 .. p - 1, each under the
        distribution behind the tokens before it (the last two None without `top`). Takes a free row and its pages
        meanwhile."""
        b = self.base
        ids = self._ids(ids)
        if ids.numel() < 2:
            raise ValueError('a text to score has at least two tokens')
        if not 1 <= rows_at_once <= 65535:
            raise ValueError('rows_at_once must be in [1, 65535]')
        row = next((r for r in range(self.batch) if not self.held[r]), None)
        if row is None:
            raise RuntimeError('no free row')
        try:
            h, _, _ = self._run([row], [ids])
        finally:
            self.release(row)
        x = ops.rmsnorm(h[:-1], b.final_norm, b.eps)
        parts = [ops.token_logprobs(_proj(x[i:i + rows_at_once], b.w_lm, b.s_lm), ids[1 + i:1 + i + rows_at_once], top=top)
                 for i in range(0, x.shape[0], rows_at_once)]
        return tuple(None if t[0] is None else torch.cat(t) for t in zip(*parts))

    # ---- steps
    def _attend_step(self, i, lay, qkv):
        b = self.base
        q, k, v = self._split(qkv)
        q = ops.kv_append_paged(k, v, self.kv[i], self.table, self.positions, q=q, **self._prologue(lay))
        return ops.attn_decode_paged(q, self.kv[i], self.table, self.positions, b.nq, b.nkv, b.d, scale=b.scale, ws=self.q8_ws)

    def _step(self):
        """The launches of a step (capturable): the next slot of every row has its page."""
        super().step()
        self.positions.masked_fill_(self.idle, -1)
        self._answer(self.logits, self.tokens)

    @torch.no_grad()
    def step(self):
        """One token for every row that has a sequence."""
        live = [r for r in range(self.batch) if self.held[r]]
        with self._all_or_nothing():
            for r in live:
                self._reserve(r, self.lengths[r] + 1)
            self._step()
            for r in live:
                self.lengths[r] += 1


class PagedGraphDecoder(RaggedGraphDecoder):
    """PagedEngine with the step captured as a CUDA graph: generate(prompts, lengths, count) -> tokens [B, count] (int64, on
    the device), or with top_logprobs (tokens, logprob [B, count], entropy [B, count], top_ids [B, count, top],
    top_logprob [B, count, top])."""

    def __init__(self, model, batch, pages, capacity, page_size=16, kv_dtype=torch.bfloat16, top_logprobs=None):
        engine = PagedEngine(model, batch, pages, capacity, page_size=page_size, kv_dtype=kv_dtype, top_logprobs=top_logprobs)
        self._init(engine)
        self.kept = []
        if engine.top is not None:  # (buffer [columns, batch, ...], the step's values)
            self.kept = [(torch.zeros((engine.cap,) + t.shape, dtype=t.dtype, device=engine.device), t)
                         for t in (engine.logprob, engine.entropy, engine.top_ids, engine.top_logprob)]

    def _park(self):
        self.engine.positions.fill_(-1)

    def _replay_body(self):
        self.engine._step()
        self.col.add_(1)
        self.out.index_copy_(1, self.col, self.engine.tokens.view(-1, 1))
        for buf, t in self.kept:
            buf.index_copy_(0, self.col, t.unsqueeze(0))

    @torch.no_grad()
    def generate(self, prompts, lengths, count):
        eng = self.engine
        check_ragged(prompts, lengths, count, eng.cap)
        if prompts.shape[0] != eng.batch:
            raise ValueError('prompts must have the decoder batch size')
        lengths = lengths.tolist()
        eng._check_anew(lengths, [n + count - 1 for n in lengths], eng.pool.pages)
        eng.reset()
        if self.graph is None:
            self._capture()
        eng.prefill(prompts, lengths)
        try:
            for r in range(eng.batch):
                eng.reserve(r, eng.lengths[r] + count - 1)
            self.col.zero_()
            self.out[:, 0] = eng.tokens
            for buf, t in self.kept:
                buf[0] = t
            for _ in range(count - 1):
                self.graph.replay()
            for r in range(eng.batch):
                eng.lengths[r] += count - 1
        except BaseException:  # an interrupt between replays: how many have run is not known
            eng.reset()
            raise
        tokens = self.out[:, :count].clone()
        if not self.kept:
            return tokens
        return (tokens,) + tuple(buf[:count].transpose(0, 1).contiguous() for buf, _ in self.kept)
