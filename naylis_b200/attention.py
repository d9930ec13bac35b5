"""Attention for serving: packed prompts, one new token over a paged cache, and
the rotary embedding that files keys and values into it (csrc/prompt.cu,
csrc/serve.cu, through the C ABI).

The training trunk attends over equal-length batches and keeps no keys; a server
prefills prompts of different lengths side by side and then extends each by one
token at a time. Per layer:

    prefill   q, k = rope_append(qkv, ...);  o = prompt_attention(q, k, v, plan)
    decode    q, _ = rope_append(qkv, ...);  o = decode_attention(q, pages, table, lens)

The cache may be held in 4 bits instead (csrc/serve_int4.cu: 9/32 of the memory and of
a step's bytes), and a step over it may bring several new tokens of a sequence, as a
check of drafted tokens does:

    prefill   q, k, v = rope_append_int4(qkv, ..., want_kv=True);  o = prompt_attention(q, k, v, plan)
    decode    q, _, _ = rope_append_int4(qkv, ...);  o = decode_attention_int4(q, *cache, table, lens)

All tensors are bf16 CUDA tensors (pages in 4 bits: uint8) with head_dim 64 or 128; a
group of query heads may share a key head. Everything else raises. Forward only: an input that requires
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


def _projection(name, qkv, cos, sin, positions, slots, H, Hk, hd):
    """The checked arguments of an append, each as the kernels take it."""
    _heads(name, hd, H, Hk)
    width = (H + 2 * Hk) * hd
    if qkv.dim() != 2 or qkv.shape[1] != width:
        raise RuntimeError(f"{name}: qkv must be (T, {width}) for {H} + 2 x {Hk} heads of {hd}, got {tuple(qkv.shape)}")
    dev, shape = qkv.device, cos.shape
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(shape) != 2 or shape[1] != hd or \
            sin.shape != shape or cos.device != dev or sin.device != dev:
        raise RuntimeError(f"{name}: cos and sin must be (n_pos, {hd}) fp32 on {dev}")
    if cos.requires_grad or sin.requires_grad:
        _no_grad(name)
    if forward_ad._current_level >= 0:
        _lib.no_tangent(name, cos, sin)
    T = qkv.shape[0]
    positions, pcode = _index(name, positions, T, dev, "positions")
    slots, scode = _index(name, slots, T, dev, "slots")
    ld, step = qkv.stride()
    if step != 1 or qkv.data_ptr() % 16 or (T > 1 and (ld % 8 or ld < width)):
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    cos, sin = cos.contiguous(), sin.contiguous()
    if cos.data_ptr() % 16:
        cos = cos.clone()
    if sin.data_ptr() % 16:
        sin = sin.clone()
    return qkv, cos, sin, positions, pcode, slots, scode


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
    qkv, cos, sin, positions, pcode, slots, scode = _projection("rope_append", qkv, cos, sin, positions, slots, H, Hk, hd)
    T, dev = qkv.shape[0], qkv.device
    q = torch.empty(T, H, hd, dtype=torch.bfloat16, device=dev)
    k = torch.empty(T, Hk, hd, dtype=torch.bfloat16, device=dev) if want_k else None
    _lib.call_on(dev.index, "mom_rope_append", qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1], cos.data_ptr(),
          sin.data_ptr(), cos.shape[0], positions.data_ptr(), pcode, slots.data_ptr(), scode, T, H, Hk, hd, P, page,
          k_pages.data_ptr(), v_pages.data_ptr(), q.data_ptr(), 0 if k is None else k.data_ptr())
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
def _block_table(name, block_table, seq_lens, B, page, max_len, dev):
    """Checked: (block_table, its pitch, seq_lens, max_len) as the kernels take them."""
    shape = block_table.shape
    if block_table.dtype != torch.int32 or len(shape) != 2 or shape[0] != B or block_table.device != dev:
        raise RuntimeError(f"{name}: block_table must be ({B}, pages) int32 on {dev}")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,) or seq_lens.device != dev:
        raise RuntimeError(f"{name}: seq_lens must be ({B},) int32 on {dev}")
    pages = table_ld = shape[1]
    if B > 1 or pages > 1:
        ld, step = block_table.stride()
        if (pages > 1 and step != 1) or (B > 1 and ld < pages):
            block_table = block_table.contiguous()
        elif B > 1:
            table_ld = ld
    seq_lens = seq_lens.contiguous()
    cap = pages * page
    max_len = cap if max_len is None else int(max_len)
    if not 0 <= max_len <= cap:
        raise RuntimeError(f"{name}: max_len {max_len} must be in [0, {cap}], what the block table holds")
    return block_table, table_ld, seq_lens, max_len


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
    block_table, table_ld, seq_lens, max_len = _block_table("decode_attention", block_table, seq_lens, B, page, max_len, dev)
    out = torch.empty(B, H, hd, dtype=torch.bfloat16, device=dev)
    need = _lib.handle().mom_decode_attn_workspace_size(B, H, Hk, hd, max_len)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call_on(dev.index, "mom_decode_attn", q.data_ptr(), q_ld, k_pages.data_ptr(), v_pages.data_ptr(), P, page,
          block_table.data_ptr(), table_ld, seq_lens.data_ptr(), max_len, B, H, Hk, hd,
          hd ** -0.5 if scale is None else float(scale), out.data_ptr(), 0 if ws is None else ws.data_ptr(), need)
    return out


# ------------------------------------------------------------------ a cache in 4 bits
GROUP = 64          # values that share a scale and a zero
MAX_NEW = 64        # new tokens of a sequence in a step


def _pages_int4(name, k_pages, v_pages, scales):
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or k_pages.dtype != torch.uint8 or v_pages.dtype != torch.uint8 or \
            not k_pages.is_cuda or v_pages.device != k_pages.device or not k_pages.is_contiguous() or \
            not v_pages.is_contiguous():
        raise RuntimeError(f"{name}: k_pages and v_pages must both be contiguous (num_pages, n_kv_heads, page_size, "
                           f"head_dim / 2) uint8 CUDA tensors, got {tuple(shape)} {k_pages.dtype} on {k_pages.device} and "
                           f"{tuple(v_pages.shape)} {v_pages.dtype} on {v_pages.device}")
    P, Hk, page, half = shape
    if page not in PAGE_SIZES:
        raise RuntimeError(f"{name}: page_size {page} must be one of {PAGE_SIZES}")
    if half not in (32, 64):
        raise RuntimeError(f"{name}: head_dim {2 * half} must be 64 or 128")
    if scales.shape != (P, Hk, page, 2 * half // GROUP, 4) or not scales.is_contiguous():
        raise RuntimeError(f"{name}: scales must be contiguous {(P, Hk, page, 2 * half // GROUP, 4)} for these pages, got "
                           f"{tuple(scales.shape)}")
    return P, Hk, page, 2 * half


def rope_append_int4(qkv, cos, sin, positions, k_pages, v_pages, scales, slots, *, n_heads: int, want_kv: bool = False):
    """rope_append into a cache in 4 bits: k_pages, v_pages (num_pages, n_kv_heads,
    page_size, hd / 2) uint8, scales (num_pages, n_kv_heads, page_size, hd / 64, 4)
    bf16, written in place.

    Each 64 values of a key (rotated, rounded to bf16) or a value keep zero = the
    least of them and scale = bf16((greatest - least) * fp32(1 / 15)), in fp32 (a product, not a
    division: the two differ where bf16 rounds a tie), and of each x the number n = round((x - zero) / scale), 0 to 15 (0 where scale is 0): it stands for
    zero + n scale. A group with a value that is not finite, or a range beyond fp32,
    stands for NaN. Two numbers share a byte, the even dimension's in the low half;
    the last axis of scales is the key's scale and zero, then the value's. Tokens of one
    call have slots of their own: of two with the same one, parts of either may be kept.

    Returns (q (T, n_heads, hd) rotated, k, v): with want_kv what the filed keys and
    values stand for, rounded to bf16, (T, n_kv_heads, hd), so that a prefill attends
    to what later steps will see; else None."""
    name = "rope_append_int4"
    P, Hk, page, hd = _pages_int4(name, k_pages, v_pages, scales)
    _check(name, qkv, scales)
    if k_pages.device != qkv.device:
        raise RuntimeError(f"{name}: tensors on {qkv.device} and {k_pages.device}")
    H = int(n_heads)
    qkv, cos, sin, positions, pcode, slots, scode = _projection(name, qkv, cos, sin, positions, slots, H, Hk, hd)
    T, dev = qkv.shape[0], qkv.device
    q = torch.empty(T, H, hd, dtype=torch.bfloat16, device=dev)
    k = torch.empty(T, Hk, hd, dtype=torch.bfloat16, device=dev) if want_kv else None
    v = torch.empty_like(k) if want_kv else None
    _lib.call_on(dev.index, "mom_rope_append_int4", qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1],
                 cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), pcode, slots.data_ptr(), scode, T, H,
                 Hk, hd, P, page, k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), q.data_ptr(),
                 0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr())
    return q, k, v


def decode_attention_int4(q, k_pages, v_pages, scales, block_table, seq_lens, *, new_lens=None, scale=None, max_len=None):
    """Attention of the newest tokens of each sequence over a cache in 4 bits: q
    (B, n, H, hd) bf16, the last n of each sequence's seq_lens keys (n at most 64), or
    with new_lens (B) int32 on the device the last new_lens of them, whose queries
    come first. New token j sees the keys 0 .. seq_len - new_len + j; one that sees none,
    and rows behind new_len, get zeros. pages and scales as rope_append_int4 files
    them; block_table, seq_lens, scale and max_len as decode_attention takes them. A
    sequence longer than max_len, with a page outside the cache or with a new_len
    outside [0, n]: NaN. What a token does not see does not reach it. A weight below
    2^-126 of its row's greatest counts as 0. Returns (B, n, H, hd) bf16."""
    name = "decode_attention_int4"
    P, Hk, page, hd = _pages_int4(name, k_pages, v_pages, scales)
    _check(name, q, scales)
    shape, dev = q.shape, q.device
    if len(shape) != 4 or shape[3] != hd:
        raise RuntimeError(f"{name}: q must be (sequences, new tokens, heads, {hd}), got {tuple(shape)}")
    if k_pages.device != dev:
        raise RuntimeError(f"{name}: tensors on {dev} and {k_pages.device}")
    B, n, H, _ = shape
    _heads(name, hd, H, Hk)
    if not 1 <= n <= MAX_NEW:
        raise RuntimeError(f"{name}: {n} new tokens must be in [1, {MAX_NEW}]")
    q_ld = H * hd
    if not q.is_contiguous() or q.data_ptr() % 16:
        q, q_ld = _rows(name, q.reshape(B * n, H, hd), "q")
    if new_lens is not None:
        if new_lens.dtype != torch.int32 or new_lens.shape != (B,) or new_lens.device != dev:
            raise RuntimeError(f"{name}: new_lens must be ({B},) int32 on {dev}")
        new_lens = new_lens.contiguous()
    block_table, table_ld, seq_lens, max_len = _block_table(name, block_table, seq_lens, B, page, max_len, dev)
    out = torch.empty(B, n, H, hd, dtype=torch.bfloat16, device=dev)
    need = _lib.handle().mom_decode_attn_int4_workspace_size(B, n, H, Hk, hd, max_len)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call_on(dev.index, "mom_decode_attn_int4", q.data_ptr(), q_ld, k_pages.data_ptr(), v_pages.data_ptr(),
                 scales.data_ptr(), P, page, block_table.data_ptr(), table_ld, seq_lens.data_ptr(),
                 0 if new_lens is None else new_lens.data_ptr(), max_len, B, n, H, Hk, hd,
                 hd ** -0.5 if scale is None else float(scale), out.data_ptr(), 0 if ws is None else ws.data_ptr(), need)
    return out


# ------------------------------------------------------------------ cache
class PagedKVCache:
    """The pages of every layer and the sequences that own them.

    k, v: (n_layers, num_pages, n_kv_heads, page_size, head_dim) bf16, or with bits 4
    (..., head_dim / 2) uint8 and scales (..., head_dim / 64, 4) bf16 (rope_append_int4's);
    layer(i) is one layer's, as the calls take them. A sequence's pages are the same in
    every layer. The book-keeping is on the host: add() a
    sequence, extend() sequences by their new tokens (which says where those go) or
    retract() those, free() one when it is done."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, *,
                 bits: int = 16, device="cuda"):
        if page_size not in PAGE_SIZES:
            raise RuntimeError(f"PagedKVCache: page_size {page_size} must be one of {PAGE_SIZES}")
        _heads("PagedKVCache", head_dim, n_kv_heads, n_kv_heads)
        if n_layers <= 0 or num_pages < 0:
            raise RuntimeError(f"PagedKVCache: {n_layers} layers of {num_pages} pages")
        if bits not in (4, 16):
            raise RuntimeError(f"PagedKVCache: {bits} bits must be 4 or 16")
        rows = (n_layers, num_pages, n_kv_heads, page_size)
        shape, dtype = (rows + (head_dim // 2,), torch.uint8) if bits == 4 else (rows + (head_dim,), torch.bfloat16)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.scales = None
        if bits == 4:
            self.scales = torch.empty(rows + (head_dim // GROUP, 4), dtype=torch.bfloat16, device=device)
        self.bits = bits
        self.page_size, self.num_pages = page_size, num_pages
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages, self._len, self._next = {}, {}, 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, i: int):
        """Layer i's pages: (k, v), and its scales with bits 4."""
        return (self.k[i], self.v[i]) if self.bits == 16 else (self.k[i], self.v[i], self.scales[i])

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


__all__ = ["GROUP", "MAX_NEW", "PAGE_SIZES", "PagedKVCache", "PromptPlan", "rope_append", "rope_append_int4",
           "prompt_attention", "decode_attention", "decode_attention_int4"]
