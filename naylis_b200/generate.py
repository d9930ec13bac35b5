"""Answering with a trained decoder: prompts of different lengths prefilled side by
side, then one token of each sequence at a time from a paged key-value cache, every
chosen token scored.

The reference's model has no cache: a new token costs a pass over its whole prefix
(model.py:350-560 runs the trunk over all positions). Here a pass over new tokens
only runs the training trunk's kernels on packed rows (csrc/trunk.cu) with

    rope_append        rotates q and k by position and files k and v into the pages
    prompt_attention   a prefill's packed sequences
    decode_attention   one new token of each sequence over its pages
    token_logprobs     the log probability, entropy and alternatives of each token

With kv_bits=4 the cache is held in 4 bits (rope_append_int4, decode_attention_int4): 9/32
of the memory and of what a step reads. A pass may append several tokens to each
sequence (Session.extend), and the last ones can be taken back (Session.retract): a
smaller model's drafts are checked together and verify_drafts says which stay.

The MoM router needs of the past only its running sum: a layer keeps, per sequence,
the fp32 prefix sum of its router input, carried in token order (the sum that the
training router's fp32 scan carries, so that a token is routed as in one pass).
Its bank's k and v are projected once.
"""
from __future__ import annotations

import dataclasses
import operator
from typing import List, Optional

import torch

from . import attention, scoring, trunk
from . import mom_kernels as mk
from .decoder import NaylisForCausalLM, rope_tables
from .sequence_parallel import CudaShardOps


@dataclasses.dataclass
class Generation:
    """One prompt's answer: its tokens, each with its log probability and the
    entropy of the distribution it was chosen from, and (top_logprobs > 0) the
    most likely alternatives there, best first."""
    tokens: List[int] = dataclasses.field(default_factory=list)
    logprobs: List[float] = dataclasses.field(default_factory=list)
    entropies: List[float] = dataclasses.field(default_factory=list)
    top_ids: List[List[int]] = dataclasses.field(default_factory=list)
    top_logprobs: List[List[float]] = dataclasses.field(default_factory=list)


def _check_model(model):
    p = model.model.embed_tokens.weight if isinstance(model, NaylisForCausalLM) else None
    if p is None or not p.is_cuda or p.dtype != torch.float32:
        raise RuntimeError("generate: a NaylisForCausalLM with fp32 parameters on a CUDA device is needed")
    cfg = model.config
    if cfg.hidden_size not in (128, 256, 512, 1024, 2048) or cfg.head_dim not in (64, 128):
        raise RuntimeError(f"generate: the serving kernels take hidden_size 128 to 2048 and head_dim 64 or 128, got "
                           f"{cfg.hidden_size} and {cfg.head_dim}")
    if cfg.scan_mode != "fp32":
        raise RuntimeError(f"generate: the carried router sum is the fp32 scan's; scan_mode is {cfg.scan_mode!r}")


class Session:
    """Sequences of one model in a paged cache, of bf16 or (kv_bits 4) of 4-bit numbers.
    add() prefills prompts, step() appends one token to each running sequence, extend()
    several; they return the next tokens' logits (rows in the order of .seqs). retract()
    takes the last tokens back, up to `undo` of a sequence; drop() ends sequences. The
    weights must not change while a session lives: the cached keys and values, and the
    bank's, projected once here, are the old ones'. An error raised by add(), step() or
    extend() leaves the session as it was."""

    def __init__(self, model: NaylisForCausalLM, num_pages: int, page_size: int = 16, kv_bits: int = 16,
                 undo: int = 0):
        _check_model(model)
        if undo < 0:
            raise RuntimeError(f"Session: undo {undo} must be >= 0")
        self.model, cfg = model, model.config
        self.device = model.model.embed_tokens.weight.device
        self.cache = attention.PagedKVCache(cfg.num_hidden_layers, num_pages, page_size, cfg.num_attention_heads,
                                            cfg.head_dim, bits=kv_bits, device=self.device)
        self.seqs: List[int] = []
        self.sums = None                 # per layer: (sequences, hidden) fp32 prefix sums of the router's input
        self.undo = undo
        self._past = None                # per layer: (sequences, undo, hidden) these sums before the last tokens
        self._known: List[int] = []      # and how many of them, from the last one back, each sequence has
        self._cos = self._sin = None
        with self._mode():
            self.bank = [trunk.bank_kv(model.model.M_blocks, l.mom.k_proj.weight, l.mom.v_proj.weight, l.mom.mem_slots)
                         for l in model.model.layers]

    def _mode(self):
        stack = torch.autocast("cuda", dtype=torch.bfloat16)
        return _NoGrad(stack)

    def _tables(self, n: int):
        if self._cos is None or self._cos.shape[0] < n:
            n = 1 << max(10, (n - 1).bit_length())
            self._cos, self._sin = rope_tables(n, self.model.config.head_dim, self.model.config.rope_theta, self.device)
        return self._cos, self._sin

    def _pass(self, ids, positions, slots, longest, attend, route, want_k):
        """The trunk over packed new tokens ids (T,): hidden states (T, hidden) bf16
        after the final norm."""
        net, cfg = self.model.model, self.model.config
        H, d = cfg.num_attention_heads, cfg.hidden_size
        cos, sin = self._tables(longest)
        x, pending = net.embed_tokens(ids), None
        for i, layer in enumerate(net.layers):
            a, m = layer.self_attn, layer.mom
            x, y = trunk.add_rmsnorm(x, pending, layer.input_layernorm.weight, layer.input_layernorm.eps)
            qkv = trunk.linear_f32grad(y, a.q_proj.weight, a.k_proj.weight, a.v_proj.weight)
            if self.cache.bits == 4:
                q, k, v = attention.rope_append_int4(qkv, cos, sin, positions, *self.cache.layer(i), slots, n_heads=H,
                                                     want_kv=want_k)
            else:
                q, k = attention.rope_append(qkv, cos, sin, positions, *self.cache.layer(i), slots, n_heads=H,
                                             want_k=want_k)
                v = qkv.view(-1, 3 * H, cfg.head_dim)[:, 2 * H:]
            o = attend(i, q, k, v)
            o = trunk.linear_f32grad(o.view(-1, d), a.o_proj.weight)
            x, y, y32 = trunk.add_rmsnorm(x, o, layer.mom_norm.weight, layer.mom_norm.eps, want_f32=True)
            idx, log_gates = route(i, m, y32)
            qm = trunk.linear_f32grad(y, m.q_proj.weight).view(1, -1, H, cfg.head_dim)
            o = mk.mom_read_log_gates(qm, *self.bank[i], idx, log_gates, num_blocks=m.num_blocks,
                                      block_size=m.block_size)
            o = trunk.linear_f32grad(o.view(-1, d), m.o_proj.weight)
            x, y = trunk.add_rmsnorm(x, o, layer.post_attention_layernorm.weight, layer.post_attention_layernorm.eps,
                                     scale=m.mom_scale)
            pending = layer.mlp(y)
        return trunk.add_rmsnorm(x, pending, net.norm.weight, net.norm.eps)[1]

    def _prefill(self, prompts, positions, slots):
        """Packed prompts through the trunk -> (hidden states, per layer prefix sums, the
        plan: its check() tells, once the caller's work is on its way, whether a wait of the
        attention gave up)."""
        lens = [len(p) for p in prompts]
        plan = attention.PromptPlan(lens, device=self.device)
        ids = torch.tensor([t for p in prompts for t in p], dtype=torch.int64, device=self.device)
        sums = []

        def attend(i, q, k, v):
            return attention.prompt_attention(q, k, v, plan)

        def route(i, m, y32):
            ops = CudaShardOps(m.router_down.weight, m.router_up.weight, m.top_blocks)
            idx, gates, ends, o = [], [], [], 0
            for n in lens:
                x = y32[None, o:o + n]
                _, top, g, end = ops.route(x, 0, ops.zero_carry(x, "fp32"), True, "fp32")
                idx.append(top)
                gates.append(g)
                ends.append(end)
                o += n
            sums.append(torch.cat(ends))
            return torch.cat(idx, 1), torch.cat(gates, 1).clamp_min(1e-9).log()

        h = self._pass(ids, positions, slots, max(lens), attend, route, True)
        return h, sums, plan

    def _check_prompts(self, prompts):
        out = [[int(t) for t in p] for p in prompts]
        V = self.model.config.vocab_size
        for p in out:
            if not p or min(p) < 0 or max(p) >= V:
                raise RuntimeError(f"generate: a prompt is one or more tokens in [0, {V})")
        return out

    def add(self, prompts):
        """Prefill prompts (lists of token ids) as new sequences; returns the logits
        (len(prompts), vocab) bf16 of each one's next token. Where it raises (the cache
        does not reach, the pass fails) nothing is added."""
        prompts = self._check_prompts(prompts)
        if not prompts:
            raise RuntimeError("generate: no prompts")
        lens = [len(p) for p in prompts]
        new = [self.cache.add() for _ in prompts]
        try:
            positions, slots = self.cache.extend(new, lens)
            with self._mode():
                h, sums, plan = self._prefill(prompts, positions, slots)
                last = torch.tensor(lens, device=self.device).cumsum(0) - 1
                logits = trunk.linear_f32grad(h[last], self.model.lm_head.weight)
            past = [s.new_zeros(len(new), self.undo, s.shape[1]) for s in sums] if self.undo else None
            if self.sums is not None:
                sums = [torch.cat(p) for p in zip(self.sums, sums)]
                past = past and [torch.cat(p) for p in zip(self._past, past)]
            plan.check()
        except BaseException:
            for s in new:
                self.cache.free(s)
            raise
        self.sums = sums
        if self.undo:
            self._past, self._known = past, self._known + [0] * len(new)
        self.seqs += new
        return logits

    def step(self, tokens):
        """Append tokens (len(self.seqs),) int32 or int64 on the device, one to each running
        sequence; returns the next logits (len(self.seqs), vocab) bf16. Where it raises
        (a token outside the vocabulary, no page left, a pass that fails) no sequence has
        grown."""
        V = self.model.config.vocab_size
        if not isinstance(tokens, torch.Tensor) or tokens.shape != (len(self.seqs),) or tokens.dtype not in (
                torch.int32, torch.int64) or tokens.device != self.device:
            raise RuntimeError(f"Session.step: tokens must be ({len(self.seqs)},) int32 or int64 on {self.device}")
        if bool(((tokens < 0) | (tokens >= V)).any()):      # the embedding would fault on them
            raise RuntimeError(f"Session.step: a token is outside [0, {V})")
        if not self.seqs:
            return torch.empty(0, V, dtype=torch.bfloat16, device=self.device)
        one = [1] * len(self.seqs)
        positions, slots = self.cache.extend(self.seqs, one)
        try:
            logits, sums = self._step(tokens, positions, slots)
            past = None
            if self.undo:
                past = [torch.cat((p[:, 1:], s[:, None]), 1) for p, s in zip(self._past, self.sums)]
        except BaseException:
            self.cache.retract(self.seqs, one)
            raise
        self.sums = sums
        if self.undo:
            self._past, self._known = past, [min(n + 1, self.undo) for n in self._known]
        return logits

    def extend(self, tokens, counts=None):
        """Append tokens[i, :counts[i]] (default: all of a row) to each running sequence;
        tokens (len(self.seqs), n) int32 or int64 on the device, counts on the host.
        Returns the logits behind each token, (len(self.seqs), n, vocab) bf16, zeros behind
        a sequence's count: what verify_drafts takes. Where it raises no sequence has
        grown."""
        V, B = self.model.config.vocab_size, len(self.seqs)
        if not isinstance(tokens, torch.Tensor) or tokens.dim() != 2 or tokens.shape[0] != B or tokens.dtype not in (
                torch.int32, torch.int64) or tokens.device != self.device:
            raise RuntimeError(f"Session.extend: tokens must be ({B}, n) int32 or int64 on {self.device}")
        n = tokens.shape[1]
        counts = [n] * B if counts is None else [operator.index(c) for c in counts]
        if len(counts) != B or any(not 0 <= c <= n for c in counts) or n > attention.MAX_NEW:
            raise RuntimeError(f"Session.extend: a count in [0, {n}] for each of {B} sequences, at most "
                               f"{attention.MAX_NEW} tokens each")
        # the places of the tokens in a (B, n) grid, and the packed ones
        at = torch.tensor([i * n + j for i, c in enumerate(counts) for j in range(c)], dtype=torch.int64,
                          device=self.device)
        ids = tokens.reshape(-1)[at]
        if bool(((ids < 0) | (ids >= V)).any()):      # the embedding would fault on them
            raise RuntimeError(f"Session.extend: a token is outside [0, {V})")
        logits = torch.zeros(B, n, V, dtype=torch.bfloat16, device=self.device)
        if not len(at):
            return logits
        positions, slots = self.cache.extend(self.seqs, counts)
        try:
            got, trail = self._extend(ids, at, n, counts, positions, slots)
            logits.view(-1, V)[at] = got
            end = torch.tensor(counts, dtype=torch.int64, device=self.device)
            sums, past = self._cut(trail, end)
        except BaseException:
            self.cache.retract(self.seqs, counts)
            raise
        self.sums = sums
        if self.undo:
            self._past, self._known = past, [min(k + c, self.undo) for k, c in zip(self._known, counts)]
        return logits

    def _extend(self, ids, at, n, counts, positions, slots):
        """extend()'s pass -> (logits of the packed tokens, per layer the router's prefix sums before
        each token of the grid and behind the last, (B, n + 1, hidden))."""
        B, even = len(counts), min(counts) == n
        table, lens, longest = self.cache.tables(self.seqs)
        new = torch.tensor(counts, dtype=torch.int32, device=self.device)
        owner, place = at // n, at % n
        sees = lens[owner] - new[owner] + place.to(torch.int32) + 1      # each token's keys
        trail = []

        def grid(x):
            if even:
                return x.view(B, n, *x.shape[1:])
            return x.new_zeros(B * n, *x.shape[1:]).index_copy_(0, at, x).view(B, n, *x.shape[1:])

        def attend(i, q, k, v):
            if self.cache.bits == 4:
                o = attention.decode_attention_int4(grid(q), *self.cache.layer(i), table, lens, new_lens=new,
                                                    max_len=longest)
                return o.view(B * n, *q.shape[1:])[at]
            # a token is a sequence of its own, of the keys that it sees
            return attention.decode_attention(q, *self.cache.layer(i), table[owner], sees, max_len=longest)

        def route(i, m, y32):
            y, steps = grid(y32), [self.sums[i]]
            for j in range(n):                     # token by token: the sums that steps of one would carry
                steps.append(steps[-1] + y[:, j])
            trail.append(torch.stack(steps, 1))
            mean = trail[-1][owner, place + 1] / sees.to(torch.float32)[:, None]
            _, idx, _, lg = mk.mom_route_log_gates(mean[:, None], m.router_down.weight, m.router_up.weight,
                                                   m.top_blocks)
            return idx.transpose(0, 1), lg.transpose(0, 1)

        with self._mode():
            h = self._pass(ids, positions, slots, longest, attend, route, False)
            return trunk.linear_f32grad(h, self.model.lm_head.weight), trail

    def _cut(self, trail, end):
        """Per layer the sums of a trail (sequences, n, hidden) at `end` of each sequence, and (undo) the
        sums before it."""
        row = torch.arange(len(end), device=self.device)
        sums = [t[row, end] for t in trail]
        if not self.undo:
            return sums, None
        u, back = self.undo, torch.arange(self.undo, device=self.device)
        past = [torch.cat((p, t), 1)[row[:, None], end[:, None] + back] for p, t in zip(self._past, trail)]
        return sums, past

    def retract(self, counts):
        """Take the last counts[i] tokens of each running sequence back, as if they had not been
        appended: at most `undo`, and no more than steps have brought since it was added. Raises,
        changing nothing, when a sequence has fewer."""
        counts = [operator.index(c) for c in counts]
        if len(counts) != len(self.seqs) or any(not 0 <= c <= k for c, k in zip(counts, self._known or [0] * len(counts))):
            raise RuntimeError(f"Session.retract: for each of {len(self.seqs)} sequences a count of tokens that can be "
                               f"taken back, at most {self._known or 0}")
        if not any(counts):
            return
        back = self.undo - torch.tensor(counts, dtype=torch.int64, device=self.device)
        row, order = torch.arange(len(counts), device=self.device), torch.arange(self.undo, device=self.device)
        trail = [torch.cat((p, s[:, None]), 1) for p, s in zip(self._past, self.sums)]
        sums = [t[row, back] for t in trail]
        past = [t[row[:, None], (order + back[:, None] - self.undo).clamp_min(0)] for t in trail]
        self.cache.retract(self.seqs, counts)
        self.sums, self._past = sums, past
        self._known = [k - c for k, c in zip(self._known, counts)]

    def _step(self, tokens, positions, slots):
        """step()'s pass -> (logits, the router's prefix sums behind it)."""
        table, lens, longest = self.cache.tables(self.seqs)
        count = lens.to(torch.float32)[:, None]
        sums = []

        def attend(i, q, k, v):
            if self.cache.bits == 4:
                return attention.decode_attention_int4(q[:, None], *self.cache.layer(i), table, lens, max_len=longest)[:, 0]
            return attention.decode_attention(q, *self.cache.layer(i), table, lens, max_len=longest)

        def route(i, m, y32):
            sums.append(self.sums[i] + y32)
            mean = sums[i] / count          # the scan's division; a sequence of one row is its own mean
            _, idx, _, lg = mk.mom_route_log_gates(mean[:, None], m.router_down.weight, m.router_up.weight,
                                                   m.top_blocks)
            return idx.transpose(0, 1), lg.transpose(0, 1)

        with self._mode():
            h = self._pass(tokens, positions, slots, longest, attend, route, False)
            return trunk.linear_f32grad(h, self.model.lm_head.weight), sums

    def drop(self, rows):
        """End the sequences at these rows of .seqs (0 .. len(.seqs) - 1) and give their pages
        back. Returns the rows that stay."""
        rows = {operator.index(i) for i in rows}
        if any(not 0 <= i < len(self.seqs) for i in rows):
            raise RuntimeError(f"Session.drop: rows {sorted(rows)} of {len(self.seqs)} sequences")
        for i in rows:
            self.cache.free(self.seqs[i])
        keep = [i for i in range(len(self.seqs)) if i not in rows]
        self.seqs = [self.seqs[i] for i in keep]
        at = torch.tensor(keep, dtype=torch.int64, device=self.device)
        if self.sums is not None:
            self.sums = [s[at] for s in self.sums]
        if self._past is not None:
            self._past = [p[at] for p in self._past]
            self._known = [self._known[i] for i in keep]
        return at


class _NoGrad:
    """no_grad and bf16 autocast together."""

    def __init__(self, autocast):
        self.autocast, self.no_grad = autocast, torch.no_grad()

    def __enter__(self):
        self.no_grad.__enter__()
        self.autocast.__enter__()

    def __exit__(self, *exc):
        self.autocast.__exit__(*exc)
        self.no_grad.__exit__(*exc)


def _choose(logits, temperature, generator):
    """The next tokens of rows of logits, greedily or sampled."""
    if temperature == 0.0:
        return logits.argmax(-1)
    return torch.multinomial(torch.softmax(logits.float() / temperature, -1), 1, generator=generator)[:, 0]


def _record(answer, tokens, scores, top_logprobs, eos_token):
    """File an answer's next tokens, up to its end; whether it has come. scores: lists of token_logprobs'."""
    for j, token in enumerate(tokens):
        answer.tokens.append(token)
        answer.logprobs.append(scores[0][j])
        answer.entropies.append(scores[1][j])
        if top_logprobs:
            answer.top_ids.append(scores[2][j])
            answer.top_logprobs.append(scores[3][j])
        if eos_token is not None and token == eos_token:
            return True
    return False


def generate(model: NaylisForCausalLM, prompts, max_new_tokens: int, *, temperature: float = 0.0,
             top_logprobs: int = 0, eos_token: Optional[int] = None, generator: Optional[torch.Generator] = None,
             page_size: int = 16, num_pages: Optional[int] = None, kv_bits: int = 16,
             draft_model: Optional[NaylisForCausalLM] = None, draft_tokens: int = 4) -> List[Generation]:
    """Continue each prompt (a list of token ids) by up to max_new_tokens, greedily
    (temperature 0, ties to the lowest id) or by sampling from
    softmax(logits / temperature), until eos_token. Scores are of the distribution
    sampled from (of softmax(logits) when greedy). num_pages sizes the cache (default:
    what the prompts and answers can take); kv_bits 4 holds it in 4 bits.

    With draft_model, a smaller model of the same vocabulary, that one drafts up to
    draft_tokens tokens at a time, which the model checks in one pass (verify_drafts): the
    answers are the model's own choices, greedily, and distributed as its own samples."""
    prompts = [list(p) for p in prompts]
    if max_new_tokens < 0 or not (temperature == 0.0 or 1e-6 <= temperature <= 1e6):
        raise RuntimeError(f"generate: max_new_tokens {max_new_tokens}, temperature {temperature}")
    if page_size not in attention.PAGE_SIZES:
        raise RuntimeError(f"generate: page_size {page_size} must be one of {attention.PAGE_SIZES}")
    if draft_model is not None:
        most = min(attention.MAX_NEW - 1, scoring.MAX_DRAFTS)
        if not 1 <= draft_tokens <= most:
            raise RuntimeError(f"generate: draft_tokens {draft_tokens} must be in [1, {most}]")
        _check_model(model)
        _check_model(draft_model)
        if draft_model.config.vocab_size != model.config.vocab_size:
            raise RuntimeError(f"generate: the draft model has {draft_model.config.vocab_size} tokens, the model "
                               f"{model.config.vocab_size}")
        if draft_model.model.embed_tokens.weight.device != model.model.embed_tokens.weight.device:
            raise RuntimeError("generate: the draft model is on another device")
    out = [Generation() for _ in prompts]
    if not prompts or max_new_tokens == 0:
        return out
    K = draft_tokens if draft_model is not None else 0
    if num_pages is None:
        num_pages = sum(-(-(len(p) + max_new_tokens) // page_size) for p in prompts)
    session = Session(model, num_pages, page_size, kv_bits=kv_bits, undo=K)
    helper = None
    if draft_model is not None:
        pages = sum(-(-(len(p) + max_new_tokens + K) // page_size) for p in prompts)
        helper = Session(draft_model, pages, page_size, kv_bits=kv_bits, undo=K)
        helper.add(prompts)
    logits = session.add(prompts)
    running = list(range(len(prompts)))
    with torch.no_grad():
        tokens = _choose(logits, temperature, generator)
        score = scoring.token_logprobs(logits, tokens, top_k=top_logprobs, temperature=temperature or 1.0)
    host = [[[x] for x in t.tolist()] for t in (tokens, *(t for t in score if t is not None))]
    while True:
        done = [i for i, r in enumerate(running) if _record(out[r], host[0][i], [t[i] for t in host[1:]], top_logprobs,
                                                             eos_token) or len(out[r].tokens) == max_new_tokens]
        if len(done) == len(running):
            return out
        if done:
            tokens = tokens[session.drop(done)]
            if helper is not None:
                helper.drop(done)
            running = [r for i, r in enumerate(running) if i not in done]
        if helper is None:
            logits = session.step(tokens)
            with torch.no_grad():
                tokens = _choose(logits, temperature, generator)
                score = scoring.token_logprobs(logits, tokens, top_k=top_logprobs, temperature=temperature or 1.0)
            host = [[[x] for x in t.tolist()] for t in (tokens, *(t for t in score if t is not None))]
        else:
            lens = [min(K, max_new_tokens - len(out[r].tokens) - 1) for r in running]
            tokens, host = _checked(session, helper, tokens, lens, K, temperature, generator, top_logprobs)


def _checked(session, helper, tokens, lens, K, temperature, generator, top_logprobs):
    """A round of drafts: the helper's up to K tokens behind `tokens`, lens of each sequence, checked by
    the session's model -> (the last token of each sequence, lists of the new tokens and their scores)."""
    steps, drafted = [tokens], []
    for _ in range(K):
        drafted.append(helper.step(steps[-1]))
        with torch.no_grad():
            steps.append(_choose(drafted[-1], temperature, generator))
    helper.step(steps[-1])                        # its keys, should all drafts stay
    logits = session.extend(torch.stack(steps, 1), [n + 1 for n in lens])
    B, V = len(lens), logits.shape[2]
    with torch.no_grad():
        u = None
        if temperature != 0.0:
            u = torch.rand(B, K + 1, generator=generator, device=session.device)
        drafts = torch.stack(steps[1:], 1)
        kept = scoring.verify_drafts(logits, drafts, u, draft_logits=torch.stack(drafted, 1) if u is not None else None,
                                     temperature=temperature,
                                     draft_lens=torch.tensor(lens, dtype=torch.int32, device=session.device))
        score = scoring.token_logprobs(logits.view(B * (K + 1), V), kept.tokens.view(-1), top_k=top_logprobs,
                                       temperature=temperature or 1.0, ignore_index=-1)
        last = kept.tokens.gather(1, kept.accepted[:, None])[:, 0]
    stay, ends = kept.accepted.tolist(), last.tolist()
    if min(ends) < 0:
        raise RuntimeError("generate: the logits are not finite")
    session.retract([n - a for n, a in zip(lens, stay)])
    helper.retract([K - a for a in stay])
    host = [kept.tokens.tolist()] + [t.view(B, K + 1, *t.shape[1:]).tolist() for t in score if t is not None]
    return last, [[row[:a + 1] for row, a in zip(rows, stay)] for rows in host]


def score(model: NaylisForCausalLM, sequences, *, top_logprobs: int = 0, temperature: float = 1.0,
          kv_bits: int = 16):
    """Log probabilities of given sequences (lists of two or more token ids) under the
    model: per sequence a scoring.TokenLogprobs of its tokens 1 .. n - 1, each given
    those before it. One packed pass; no cache (kv_bits 4: its keys and values are rounded
    as one in 4 bits would)."""
    session = Session(model, 0, 16, kv_bits)
    sequences = session._check_prompts(sequences)
    if any(len(s) < 2 for s in sequences):
        raise RuntimeError("score: a sequence is two or more tokens")
    if not sequences:
        return []
    lens = [len(s) for s in sequences]
    positions = torch.cat([torch.arange(n) for n in lens]).to(session.device)
    slots = torch.full_like(positions, -1)
    with session._mode():
        h, _, plan = session._prefill(sequences, positions, slots)
        logits = trunk.linear_f32grad(h, model.lm_head.weight)
        targets = torch.tensor([t for s in sequences for t in s[1:] + [-100]], device=session.device)
        r = scoring.token_logprobs(logits, targets, top_k=top_logprobs, temperature=temperature)
    plan.check()
    out, o = [], 0
    for n in lens:
        out.append(scoring.TokenLogprobs(*(None if t is None else t[o:o + n - 1] for t in r)))
        o += n
    return out


__all__ = ["Generation", "Session", "generate", "score"]
