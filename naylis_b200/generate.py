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
    """Sequences of one model in a paged cache. add() prefills prompts, step()
    appends one token to each running sequence; both return the next token's logits
    (rows in the order of .seqs). drop() ends sequences. The weights must not change
    while a session lives: the cached keys and values, and the bank's, projected once
    here, are the old ones'. An error raised by add() or step() leaves the session as
    it was."""

    def __init__(self, model: NaylisForCausalLM, num_pages: int, page_size: int = 16):
        _check_model(model)
        self.model, cfg = model, model.config
        self.device = model.model.embed_tokens.weight.device
        self.cache = attention.PagedKVCache(cfg.num_hidden_layers, num_pages, page_size, cfg.num_attention_heads,
                                            cfg.head_dim, device=self.device)
        self.seqs: List[int] = []
        self.sums = None                 # per layer: (sequences, hidden) fp32 prefix sums of the router's input
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
            q, k = attention.rope_append(qkv, cos, sin, positions, self.cache.k[i], self.cache.v[i], slots, n_heads=H,
                                         want_k=want_k)
            o = attend(i, q, k, qkv.view(-1, 3 * H, cfg.head_dim)[:, 2 * H:])
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
            plan.check()
        except BaseException:
            for s in new:
                self.cache.free(s)
            raise
        self.sums = sums if self.sums is None else [torch.cat(p) for p in zip(self.sums, sums)]
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
        except BaseException:
            self.cache.retract(self.seqs, one)
            raise
        self.sums = sums
        return logits

    def _step(self, tokens, positions, slots):
        """step()'s pass -> (logits, the router's prefix sums behind it)."""
        table, lens, longest = self.cache.tables(self.seqs)
        count = lens.to(torch.float32)[:, None]
        sums = []

        def attend(i, q, k, v):
            return attention.decode_attention(q, self.cache.k[i], self.cache.v[i], table, lens, max_len=longest)

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


def generate(model: NaylisForCausalLM, prompts, max_new_tokens: int, *, temperature: float = 0.0,
             top_logprobs: int = 0, eos_token: Optional[int] = None, generator: Optional[torch.Generator] = None,
             page_size: int = 16, num_pages: Optional[int] = None) -> List[Generation]:
    """Continue each prompt (a list of token ids) by up to max_new_tokens, greedily
    (temperature 0, ties to the lowest id) or by sampling from
    softmax(logits / temperature), until eos_token. Scores are of the distribution
    sampled from (of softmax(logits) when greedy). num_pages sizes the cache (default:
    what the prompts and answers can take)."""
    prompts = [list(p) for p in prompts]
    if max_new_tokens < 0 or not (temperature == 0.0 or 1e-6 <= temperature <= 1e6):
        raise RuntimeError(f"generate: max_new_tokens {max_new_tokens}, temperature {temperature}")
    if page_size not in attention.PAGE_SIZES:
        raise RuntimeError(f"generate: page_size {page_size} must be one of {attention.PAGE_SIZES}")
    out = [Generation() for _ in prompts]
    if not prompts or max_new_tokens == 0:
        return out
    if num_pages is None:
        num_pages = sum(-(-(len(p) + max_new_tokens) // page_size) for p in prompts)
    session = Session(model, num_pages, page_size)
    logits = session.add(prompts)
    running = list(range(len(prompts)))
    for n in range(max_new_tokens):
        with torch.no_grad():
            if temperature == 0.0:
                tokens = logits.argmax(-1)
            else:
                tokens = torch.multinomial(torch.softmax(logits.float() / temperature, -1), 1,
                                           generator=generator)[:, 0]
            score = scoring.token_logprobs(logits, tokens, top_k=top_logprobs, temperature=temperature or 1.0)
        host = [t if t is None else t.tolist() for t in (tokens, *score)]
        done = []
        for i, r in enumerate(running):
            g = out[r]
            g.tokens.append(host[0][i])
            g.logprobs.append(host[1][i])
            g.entropies.append(host[2][i])
            if top_logprobs:
                g.top_ids.append(host[3][i])
                g.top_logprobs.append(host[4][i])
            if eos_token is not None and host[0][i] == eos_token:
                done.append(i)
        if n + 1 == max_new_tokens or len(done) == len(running):
            break
        if done:
            tokens = tokens[session.drop(done)]
            running = [r for i, r in enumerate(running) if i not in done]
        logits = session.step(tokens)
    return out


def score(model: NaylisForCausalLM, sequences, *, top_logprobs: int = 0, temperature: float = 1.0):
    """Log probabilities of given sequences (lists of two or more token ids) under the
    model: per sequence a scoring.TokenLogprobs of its tokens 1 .. n - 1, each given
    those before it. One packed pass; no cache."""
    session = Session(model, 0)
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
