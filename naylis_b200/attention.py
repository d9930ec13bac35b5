"""Attention for serving: packed prompts, one new token over a paged cache, and
the rotary embedding that files keys and values into it (csrc/prompt.cu,
csrc/serve.cu, through the C ABI).

The training trunk attends over equal-length batches and keeps no keys; a server
prefills prompts of different lengths side by side and then extends each by one
token at a time. Per layer:

    prefill   q, k = rope_append(qkv, ...);  o = prompt_attention(q, k, v, plan)
    decode    q, _ = rope_append(qkv, ...);  o = decode_attention(q, pages, table, lens)

All tensors are bf16 CUDA tensors with head_dim 64 or 128; a group of query heads
may share a key head. Everything else raises. Forward only: an input that requires
grad raises while grad mode is on (training attends through torch's attention).
"""
from __future__ import annotations

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

PAGE_SIZES = (8, 16, 32, 64, 128, 256)


def _check(name, *ts):
    dev = ts[0].device
    for t in ts:
        if t.dtype != torch.bfloat16 or not t.is_cuda:
            raise RuntimeError(f"{name} takes bf16 CUDA tensors, got {t.dtype} on {t.device}")
        if t.device != dev:
            raise RuntimeError(f"{name}: tensors on {dev} and {t.device}")
        if t.requires_grad:
            _no_grad(name)
    if forward_ad._current_level >= 0:
        _lib.no_tangent(name, *ts)


def _no_grad(name):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} is forward only: run it under torch.no_grad() or detach its inputs")


def _rows(name, t, what):
    """A (T, heads, hd) tensor whose rows hold their heads side by side, 16-byte
    aligned: itself when its strides allow (a slice of a fused projection's
    output), else a copy."""
    if t.dim() != 3:
        raise RuntimeError(f"{name}: {what} must be (tokens, heads, head_dim), got {tuple(t.shape)}")
    T, H, hd = t.shape
    if t.is_contiguous():
        if t.data_ptr() % 16 == 0:
            return t, H * hd
        return t.clone(), H * hd
    ld, sh, sd = t.stride()
    if sd == 1 and (sh == hd or H == 1) and t.data_ptr() % 16 == 0 and (T <= 1 or (ld % 8 == 0 and ld >= H * hd)):
        return t, ld if T > 1 else H * hd
    t = t.contiguous()
    return (t if t.data_ptr() % 16 == 0 else t.clone()), H * hd


def _pages(name, k_pages, v_pages):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise RuntimeError(f"{name}: k_pages and v_pages must both be (num_pages, n_kv_heads, page_size, head_dim), "
                           f"got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise RuntimeError(f"{name}: k_pages and v_pages must be contiguous")
    if k_pages.shape[2] not in PAGE_SIZES:
        raise RuntimeError(f"{name}: page_size {k_pages.shape[2]} must be one of {PAGE_SIZES}")


def _index(name, t, n, dev, what):
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (n,) or t.device != dev:
        raise RuntimeError(f"{name}: {what} must be ({n},) int32 or int64 on {dev}, got {tuple(t.shape)} {t.dtype} "
                           f"on {t.device}")
    return t.contiguous(), _lib.I32 if t.dtype == torch.int32 else _lib.I64


def _heads(name, hd, H, Hk):
    if hd not in (64, 128):
        raise RuntimeError(f"{name}: head_dim {hd} must be 64 or 128")
    if H <= 0 or Hk <= 0 or H % Hk:
        raise RuntimeError(f"{name}: {H} query heads are not a multiple of {Hk} key heads")


# ------------------------------------------------------------------ cache write
def rope_append(qkv, cos, sin, positions, k_pages, v_pages, slots, *, n_heads: int, want_k: bool = False):
    """Rotate the heads of a fused projection by their tokens' positions and file
    the keys and values into the cache.

    qkv (T, (n_heads + 2 n_kv_heads) * hd) bf16: [q | k | v] heads of each token
    (n_kv_heads and hd are the cache's); cos, sin (n_pos, hd) fp32 (rope_tables);
    positions (T) the row of the tables, slots (T) page * page_size + offset, both
    int32 or int64; k_pages, v_pages (num_pages, n_kv_heads, page_size, hd),
    written in place. A slot outside the cache is not written (-1: padding); a
    position outside the tables makes the token's q and k NaN; two tokens must not
    share a slot. Returns (q (T, n_heads, hd) rotated, k (T, n_kv_heads, hd)
    rotated if want_k else None). The values stay where they are:
    qkv.view(T, -1, hd)[:, n_heads + n_kv_heads:]."""
    _check("rope_append", qkv, k_pages, v_pages)
    _pages("rope_append", k_pages, v_pages)
    P, Hk, page, hd = k_pages.shape
    H = int(n_heads)
    _heads("rope_append", hd, H, Hk)
    if qkv.dim() != 2 or qkv.shape[1] != (H + 2 * Hk) * hd:
        raise RuntimeError(f"rope_append: qkv must be (T, {(H + 2 * Hk) * hd}) for {H} + 2 x {Hk} heads of {hd}, got "
                           f"{tuple(qkv.shape)}")
    dev = qkv.device
    for t in (cos, sin):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != hd or t.shape != cos.shape or t.device != dev:
            raise RuntimeError(f"rope_append: cos and sin must be (n_pos, {hd}) fp32 on {dev}")
        if t.requires_grad:
            _no_grad("rope_append")
    if forward_ad._current_level >= 0:
        _lib.no_tangent("rope_append", cos, sin)
    T = qkv.shape[0]
    positions, pcode = _index("rope_append", positions, T, dev, "positions")
    slots, scode = _index("rope_append", slots, T, dev, "slots")
    if qkv.stride(1) != 1 or qkv.data_ptr() % 16 or (T > 1 and (qkv.stride(0) % 8 or qkv.stride(0) < qkv.shape[1])):
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    cos, sin = cos.contiguous(), sin.contiguous()
    if cos.data_ptr() % 16:
        cos = cos.clone()
    if sin.data_ptr() % 16:
        sin = sin.clone()
    q = torch.empty(T, H, hd, dtype=torch.bfloat16, device=dev)
    k = torch.empty(T, Hk, hd, dtype=torch.bfloat16, device=dev) if want_k else None
    _lib.call_on(dev.index, "mom_rope_append", qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1], cos.data_ptr(),
          sin.data_ptr(), cos.shape[0], positions.data_ptr(), pcode, slots.data_ptr(), scode, T, H, Hk, hd, P, page,
          k_pages.data_ptr(), v_pages.data_ptr(), q.data_ptr(), None if k is None else k.data_ptr())
    return q, k


# ------------------------------------------------------------------ prompts
class PromptPlan:
    """The work list of prompt_attention for one batch of lengths; it holds for
    every layer. q_lens: query tokens of each sequence, in packed order; k_lens:
    its keys (default: the same), the queries being its last ones. The list for a
    pair of head counts is made when it is first asked for."""

    def __init__(self, q_lens, k_lens=None, *, device="cuda"):
        self.q_lens = tuple(int(n) for n in q_lens)
        self.k_lens = self.q_lens if k_lens is None else tuple(int(n) for n in k_lens)
        if len(self.k_lens) != len(self.q_lens):
            raise RuntimeError(f"PromptPlan: {len(self.q_lens)} query lengths and {len(self.k_lens)} key lengths")
        top = 1 << 30
        if any(not 0 <= n <= top for n in self.q_lens + self.k_lens) or sum(self.q_lens) > top or \
                sum(self.k_lens) > top:
            raise RuntimeError("PromptPlan: lengths, and their sums, must be in [0, 2^30]")
        self.total_q, self.total_k = sum(self.q_lens), sum(self.k_lens)
        self.device = torch.empty(0, device=device).device
        self._lists = {}      # by head counts: the buffer, the stream that it was made on

    def list_for(self, n_heads: int, n_kv_heads: int):
        """The device buffer of the work list for these head counts. The first call copies it
        from the host, which a graph capture refuses: ask, or run a call, before one."""
        got, own = self._lists.get((n_heads, n_kv_heads), (None, 0))
        stream = torch._C._cuda_getCurrentRawStream(self.device.index) if self.device.type == "cuda" else 0
        if got is None:
            n = len(self.q_lens)
            lens = np.asarray(self.q_lens + self.k_lens + (0,), dtype=np.int64)
            ql, kl = lens.ctypes.data, lens.ctypes.data + 8 * n
            size = _lib.load().mom_prompt_plan_size(ql, n, n_heads, n_kv_heads)
            if size == 0:
                raise RuntimeError(f"PromptPlan: {_lib.last_error()}")
            host = torch.empty(size, dtype=torch.uint8)
            _lib.call("mom_prompt_plan", ql, kl, n, n_heads, n_kv_heads, host.data_ptr(), size)
            got, own = self._lists[n_heads, n_kv_heads] = host.to(self.device), stream
        if stream != own:      # the list lives until the work of every stream that asks for it is done
            got.record_stream(torch.cuda.current_stream(self.device))
        return got

    def check(self):
        """Raise if a kernel that used this plan gave up a wait: of the work before it on the
        current stream, which it synchronises."""
        for buffer, _ in self._lists.values():
            _lib.call_on(self.device.index, "mom_prompt_plan_check", buffer.data_ptr())


def prompt_attention(q, k, v, plan: PromptPlan, *, scale=None):
    """Causal attention over packed prompts: q (Tq, H, hd), k and v (Tk, Hk, hd)
    bf16, the plan's sequences one after another (token strides may be a fused
    projection's); query head h reads key head h // (H // Hk). Row r of a sequence
    of Lq queries and Lk keys sees its keys 0 .. Lk - Lq + r; one that sees none
    gets zeros. scale (> 0) defaults to hd ** -0.5. Returns (Tq, H, hd) bf16."""
    _check("prompt_attention", q, k, v)
    q, q_ld = _rows("prompt_attention", q, "q")
    k, k_ld = _rows("prompt_attention", k, "k")
    v, v_ld = _rows("prompt_attention", v, "v")
    Tq, H, hd = q.shape
    Tk, Hk, _ = k.shape
    if k.shape != v.shape or k.shape[2] != hd:
        raise RuntimeError(f"prompt_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    _heads("prompt_attention", hd, H, Hk)
    if Tq != plan.total_q or Tk != plan.total_k:
        raise RuntimeError(f"prompt_attention: {Tq} queries and {Tk} keys, the plan has {plan.total_q} and "
                           f"{plan.total_k}")
    if plan.device != q.device:
        raise RuntimeError(f"prompt_attention: the plan is on {plan.device}, q on {q.device}")
    out = torch.empty(Tq, H, hd, dtype=torch.bfloat16, device=q.device)
    work = plan.list_for(H, Hk)
    _lib.call_on(q.device.index, "mom_prompt_attn", q.data_ptr(), q_ld, k.data_ptr(), k_ld, v.data_ptr(), v_ld, Tq, Tk,
                 H, Hk, hd, hd ** -0.5 if scale is None else float(scale), work.data_ptr(), work.numel(), out.data_ptr())
    return out


# ------------------------------------------------------------------ decode
def decode_attention(q, k_pages, v_pages, block_table, seq_lens, *, scale=None, max_len=None):
    """Attention of one new token per sequence over its cached keys: q (B, H, hd)
    bf16; k_pages, v_pages (num_pages, Hk, page_size, hd); block_table (B, n)
    int32, each sequence's pages in order; seq_lens (B) int32 on the device, each
    sequence's keys (the new token's among them). max_len, known to the host,
    bounds seq_lens (default n * page_size); the keys are shared out by the lengths
    themselves, so it need not be near. A sequence of length <= 0 gets zeros; one
    longer than max_len, or with a page outside the cache, NaN. Returns (B, H, hd)
    bf16."""
    _check("decode_attention", q, k_pages, v_pages)
    _pages("decode_attention", k_pages, v_pages)
    q, q_ld = _rows("decode_attention", q, "q")
    B, H, hd = q.shape
    P, Hk, page, hd_k = k_pages.shape
    if hd_k != hd:
        raise RuntimeError(f"decode_attention: q has head_dim {hd}, the cache {hd_k}")
    _heads("decode_attention", hd, H, Hk)
    dev = q.device
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or \
            block_table.device != dev:
        raise RuntimeError(f"decode_attention: block_table must be ({B}, pages) int32 on {dev}")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,) or seq_lens.device != dev:
        raise RuntimeError(f"decode_attention: seq_lens must be ({B},) int32 on {dev}")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    seq_lens = seq_lens.contiguous()
    table_ld = block_table.stride(0) if B > 1 else block_table.shape[1]
    if table_ld < block_table.shape[1]:
        block_table = block_table.contiguous()
        table_ld = block_table.shape[1]
    cap = block_table.shape[1] * page
    max_len = cap if max_len is None else int(max_len)
    if not 0 <= max_len <= cap:
        raise RuntimeError(f"decode_attention: max_len {max_len} must be in [0, {cap}], what the block table holds")
    out = torch.empty(B, H, hd, dtype=torch.bfloat16, device=dev)
    need = _lib.load().mom_decode_attn_workspace_size(B, H, Hk, hd, max_len)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call_on(dev.index, "mom_decode_attn", q.data_ptr(), q_ld, k_pages.data_ptr(), v_pages.data_ptr(), P, page,
          block_table.data_ptr(), table_ld, seq_lens.data_ptr(), max_len, B, H, Hk, hd,
          hd ** -0.5 if scale is None else float(scale), out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    return out


# ------------------------------------------------------------------ cache
class PagedKVCache:
    """The pages of every layer and the sequences that own them.

    k, v: (n_layers, num_pages, n_kv_heads, page_size, head_dim) bf16; a sequence's
    pages are the same in every layer. The book-keeping is on the host: add() a
    sequence, extend() sequences by their new tokens (which says where those go) or
    retract() those, free() one when it is done."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, *,
                 device="cuda"):
        if page_size not in PAGE_SIZES:
            raise RuntimeError(f"PagedKVCache: page_size {page_size} must be one of {PAGE_SIZES}")
        _heads("PagedKVCache", head_dim, n_kv_heads, n_kv_heads)
        if n_layers <= 0 or num_pages < 0:
            raise RuntimeError(f"PagedKVCache: {n_layers} layers of {num_pages} pages")
        shape = (n_layers, num_pages, n_kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.page_size, self.num_pages = page_size, num_pages
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages, self._len, self._next = {}, {}, 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._len[seq]

    def add(self) -> int:
        """A new sequence without tokens."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def free(self, seq: int) -> None:
        """Give a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq]

    def extend(self, seqs, counts):
        """Room for counts[i] more tokens of seqs[i] (each named once). Returns
        (positions, slots) of the new tokens, packed in that order, int64 on the
        device: rope_append's arguments. Raises, changing nothing, when the pages do
        not reach."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise RuntimeError("PagedKVCache.extend: one count >= 0 for each sequence, each named once")
        page = self.page_size
        need = [-(-(self._len[s] + c) // page) - len(self._pages[s]) for s, c in zip(seqs, counts)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(need)} pages needed, {len(self._free)} of {self.num_pages} free")
        pos, slots = [], []
        for s, c, n in zip(seqs, counts, need):
            pages = self._pages[s]
            pages.extend(self._free.pop() for _ in range(n))
            at = np.arange(self._len[s], self._len[s] + c, dtype=np.int64)
            pos.append(at)
            slots.append(np.asarray(pages, dtype=np.int64)[at // page] * page + at % page if c else at)
            self._len[s] += c
        if not pos:
            both = np.zeros((2, 0), dtype=np.int64)
        else:
            both = np.stack([np.concatenate(pos), np.concatenate(slots)])
        both = torch.from_numpy(both).to(self.k.device)
        return both[0], both[1]

    def retract(self, seqs, counts):
        """Take the last counts[i] tokens of seqs[i] (each named once) back: what undoes an
        extend() whose pass failed. Raises, changing nothing, when one has fewer."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(
                not 0 <= c <= self._len[s] for s, c in zip(seqs, counts)):
            raise RuntimeError("PagedKVCache.retract: one count in [0, length] for each sequence, each named once")
        for s, c in zip(reversed(seqs), reversed(counts)):
            self._len[s] -= c
            pages, keep = self._pages[s], -(-self._len[s] // self.page_size)
            self._free.extend(reversed(pages[keep:]))
            del pages[keep:]

    def tables(self, seqs):
        """(block_table (B, n), seq_lens (B)) int32 on the device, and the longest
        length: decode_attention's arguments."""
        seqs = list(seqs)
        most = max((len(self._pages[s]) for s in seqs), default=0)
        table = np.zeros((len(seqs), most + 1), dtype=np.int32)
        for i, s in enumerate(seqs):
            table[i, 0] = self._len[s]
            table[i, 1:1 + len(self._pages[s])] = self._pages[s]
        both = torch.from_numpy(table).to(self.k.device)
        return both[:, 1:], both[:, 0].contiguous(), max((self._len[s] for s in seqs), default=0)


__all__ = ["PAGE_SIZES", "PagedKVCache", "PromptPlan", "rope_append", "prompt_attention", "decode_attention"]
