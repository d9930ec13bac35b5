"""The operators of a 4-bit cache and of drafted tokens, as a user calls them, next to their plain forms.

``rope_append_int4`` rotates a projection's heads and files keys and values into a
paged cache in 4 bits, ``decode_attention_int4`` attends one or several new tokens
of each sequence over that cache, ``verify_drafts`` decides which drafted tokens the
target's distribution keeps and draws the token that follows them.

A row of the cache (a token's key or value of one head) is cut into groups of 64
values. A group keeps zero = its least value and scale = bf16((greatest - least) / 15),
and of each value x the number n = round((x - zero) / scale), 0 to 15; it stands for
zero + n scale. Two numbers share a byte, the even dimension's in the low half.

A case is a dict of plain values. Sequence lengths of a batch are spread from
its ``longest`` down by ``lengths`` below, so a case names them by three numbers.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
GROUP = 64


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's keys and values of 48 sequences, the decoder's own heads
        {"name": "append-step-48", "op": "append", "seqs": 48, "longest": 1, "spread": 1.0, "past": 1500,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16},
        # a round of drafted tokens: 7 of each of 33 sequences, grouped heads of 128
        {"name": "append-drafts-33x7", "op": "append", "seqs": 33, "longest": 7, "spread": 1.0, "past": 4093,
         "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 32},
        # a prefill's 16 thousand tokens
        {"name": "append-prompt-8x2048", "op": "append", "seqs": 8, "longest": 2048, "spread": 1.0, "past": 0,
         "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 64},
        # one user's next token: latency
        {"name": "decode-one-577", "op": "decode", "seqs": 1, "longest": 577, "spread": 1.0, "new": 1,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16},
        # a batch of conversations of very different lengths, the decoder's own heads
        {"name": "decode-48-ragged", "op": "decode", "seqs": 48, "longest": 4096, "spread": 64.0, "new": 1,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 32},
        # a step that checks four drafted tokens of each sequence, grouped heads
        {"name": "decode-24x5-drafts", "op": "decode", "seqs": 24, "longest": 8191, "spread": 8.0, "new": 5,
         "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 16},
        # a few long documents, grouped heads
        {"name": "decode-4x131072", "op": "decode", "seqs": 4, "longest": 131072, "spread": 1.5, "new": 1,
         "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 64},
        # many long conversations, one head of keys for each head of queries
        {"name": "decode-16x32768", "op": "decode", "seqs": 16, "longest": 32768, "spread": 1.0, "new": 1,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 64},
        # one user's four drafts, sampled: latency
        {"name": "verify-one-4", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "dtype": "bfloat16",
         "mode": "sampled", "temperature": 1.0},
        # a busy server's drafts from a smaller model
        {"name": "verify-48x4", "op": "verify", "seqs": 48, "drafts": 4, "vocab": 32000, "dtype": "bfloat16",
         "mode": "sampled", "temperature": 0.8},
        # drafts looked up in the prompt (no distribution of their own), an odd vocabulary in fp32
        {"name": "verify-lookup-odd", "op": "verify", "seqs": 40, "drafts": 7, "vocab": 32003, "dtype": "float32",
         "mode": "lookup", "temperature": 1.0},
        # a large batch, answered greedily
        {"name": "verify-greedy-256x7", "op": "verify", "seqs": 256, "drafts": 7, "vocab": 32000, "dtype": "bfloat16",
         "mode": "greedy", "temperature": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "verify"])
    if op == "verify":
        c = {"op": op, "vocab": _log_int(rng, 2, 65000), "dtype": rng.choice(["bfloat16", "float32"]),
             "mode": rng.choice(["sampled", "sampled", "lookup", "greedy"]), "drafts": rng.randint(1, 8)}
        c["temperature"] = 0.0 if c["mode"] == "greedy" else rng.choice([1.0, 1.0, 0.7, 1.3])
        c["seqs"] = _log_int(rng, 1, max(1, min(256, 192 * 8 * 32000 // (4 * c["vocab"] * c["drafts"]))))
        return c
    c = {"op": op, "head_dim": rng.choice([64, 128]), "kv_heads": rng.choice([1, 2, 4, 8, 16])}
    c["heads"] = c["kv_heads"] * rng.choice([g for g in (1, 2, 4, 5, 8, 16) if g * c["kv_heads"] <= 32])
    c["seqs"] = _log_int(rng, 1, 64)
    c["spread"] = rng.choice([1.0, 1.5, 8.0, 100.0])
    c["page"] = rng.choice([8, 16, 32, 64, 128])
    if op == "append":
        c["past"] = rng.choice([0, _log_int(rng, 1, 4096)])
        c["longest"] = _log_int(rng, 1, max(1, min(8192, 8 * 2048 * 24 * 128 // (
            c["seqs"] * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]))))
        return c
    c["new"] = rng.choice([1, 1, 2, 3, 5, 8])
    most = 16 * 32768 * 16 * 64 // (2 * c["seqs"] * c["kv_heads"] * c["head_dim"] * (1 if c["new"] == 1 else 2))
    c["longest"] = max(c["new"], _log_int(rng, 1, max(1, min(131072, most))))
    return c


def lengths(case):
    """The batch's lengths: from `longest` down to longest / spread, evenly in the logarithm, in a mixed order."""
    n, hi = case["seqs"], case["longest"]
    lo = max(1.0, hi / case["spread"])
    got = [hi if n == 1 else max(1, int(round(hi * (lo / hi) ** (i / (n - 1))))) for i in range(n)]
    return [int(got[i]) for i in np.random.RandomState(7).permutation(n)]


def new_tokens(case):
    """New tokens of each sequence: `new`, or fewer for every fifth one and where the sequence is shorter."""
    return [min(n, case["new"] if i % 5 != 3 else max(1, case["new"] // 2)) for i, n in enumerate(lengths(case))]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 26):      # bounded fp32 temporaries
        n = min(1 << 26, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=DEV) * scale
    return out


def _table(case, lens, seed):
    """Every sequence's pages scattered over the pool, as after long use. -> (pages, table)"""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(int(seed)))
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    o = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[o:o + n].to(torch.int32)
        o += n
    return total, table


def _nibbles(g, *shape):
    """Pages as normal keys and values leave them: numbers around the middle of their groups."""
    out = torch.empty(shape, dtype=torch.uint8, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 25):
        n = min(1 << 25, flat.numel() - i)
        a = (torch.randn(2 * n, generator=g, device=DEV) * 3.2 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        flat[i:i + n] = a[0::2] | a[1::2] << 4
    return out


def _cache(case, total, g):
    Hk, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    k, v = _nibbles(g, total, Hk, page, hd // 2), _nibbles(g, total, Hk, page, hd // 2)
    scales = torch.empty(total, Hk, page, hd // GROUP, 4, dtype=torch.bfloat16, device=DEV)
    step = 0.31 * (1 + 0.1 * torch.randn(*scales.shape[:-1], 2, generator=g, device=DEV)).clamp_min(0.3)
    scales[..., 0::2] = step                                                            # of the key, of the value
    scales[..., 1::2] = -7.5 * step + 0.1 * torch.randn(step.shape, generator=g, device=DEV)      # their zeros
    return k, v, scales


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "verify":
        return _prepare_verify(case, g)
    H, Hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lens = lengths(case)
    st = {"case": case, "lens": lens, "scale": hd ** -0.5}
    if op == "decode":
        total, table = _table(case, lens, seed)
        st["q"] = _randn(g, len(lens), case["new"], H, hd, scale=2.0)
        st["k_pages"], st["v_pages"], st["scales"] = _cache(case, total, g)
        st["table"] = table.to(DEV)
        st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["new"] = new_tokens(case)
        if case["new"] > 1:
            st["new_lens"] = torch.tensor(st["new"], dtype=torch.int32, device=DEV)
        return st
    past = case["past"]
    full = [n + past for n in lens]
    total, table = _table(case, full, seed)
    T = sum(lens)
    st["qkv"] = _randn(g, T, (H + 2 * Hk) * hd)
    inv = 1.0 / (500000.0 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd))
    ang = torch.outer(torch.arange(max(full), device=DEV, dtype=torch.float64), inv)
    st["cos"] = torch.cat((ang, ang), 1).cos().float()
    st["sin"] = torch.cat((ang, ang), 1).sin().float()
    pos = torch.cat([torch.arange(past, past + n) for n in lens])
    row = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])
    st["positions"] = pos.to(DEV)
    st["slots"] = (table[row, pos // case["page"]].long() * case["page"] + pos % case["page"]).to(DEV)
    st["k_pages"], st["v_pages"], st["scales"] = _cache(case, total, g)
    return st


def _prepare_verify(case, g):
    B, K, V, mode, T = case["seqs"], case["drafts"], case["vocab"], case["mode"], case["temperature"]
    dt = getattr(torch, case["dtype"])
    # an LM head's logits: a few units wide, with some clear favourites
    logits = _randn(g, B, K + 1, V, scale=2.0, dtype=dt)
    fav = torch.randint(0, V, (B, K + 1, 4), generator=g, device=DEV)
    logits.scatter_(2, fav, (9.0 + 3.0 * torch.rand(B, K + 1, 4, generator=g, device=DEV)).to(dt))
    st = {"case": case, "logits": logits, "uniforms": None, "draft_logits": None}
    if mode == "lookup":
        pick = torch.rand(B, K, generator=g, device=DEV) < 0.7
        st["drafts"] = torch.where(pick, fav[:, :K, 0], torch.randint(0, V, (B, K), generator=g, device=DEV))
    else:
        # a smaller model's: the target's with noise, its drafts from its own distribution
        draft = torch.empty(B, K, V, dtype=dt, device=DEV)
        st["drafts"] = torch.empty(B, K, dtype=torch.int64, device=DEV)
        for b in range(0, B, 16):
            x = logits[b:b + 16, :K].float() + 0.5 * torch.randn(min(16, B - b), K, V, generator=g, device=DEV)
            draft[b:b + 16] = x
            x = draft[b:b + 16].float()
            if T > 0:
                x = x / T - torch.log(-torch.log(torch.rand(x.shape, generator=g, device=DEV).clamp(1e-9, 1 - 1e-6)))
            st["drafts"][b:b + 16] = x.argmax(-1)
        if mode == "sampled":
            st["draft_logits"] = draft
    if mode != "greedy":
        st["uniforms"] = torch.rand(B, K + 1, generator=g, device=DEV)
    short = torch.rand(B, generator=g, device=DEV) < 0.2           # sequences with fewer drafts than the others
    st["draft_lens"] = torch.where(short, torch.randint(0, K + 1, (B,), generator=g, device=DEV),
                                   K).to(torch.int32)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    return {"append": _run_append, "decode": _run_decode, "verify": _run_verify}[state["case"]["op"]](state)


def _to_4bit(x):
    """x (..., hd) bf16 -> numbers (..., hd) uint8, scale and zero (..., groups) fp32."""
    y = x.float().unflatten(-1, (-1, GROUP))
    zero = y.amin(-1, keepdim=True)
    step = ((y.amax(-1, keepdim=True) - zero) * (1.0 / 15.0)).bfloat16().float()
    n = torch.where(step > 0, (y - zero) / step, 0.0).round().clamp(0, 15)
    return n.flatten(-2).to(torch.uint8), step[..., 0], zero[..., 0]


def _from_4bit(n, step, zero):
    return (n.unflatten(-1, (-1, GROUP)).float() * step.unsqueeze(-1) + zero.unsqueeze(-1)).flatten(-2)


def _run_append(st):
    case = st["case"]
    H, Hk, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    kp, vp, scales = st["k_pages"], st["v_pages"], st["scales"]
    if own:
        from naylis_b200 import attention
        q, k, v = attention.rope_append_int4(st["qkv"], st["cos"], st["sin"], st["positions"], kp, vp, scales,
                                             st["slots"], n_heads=H, want_kv=True)
    else:
        x = st["qkv"].view(-1, H + 2 * Hk, hd)
        cos, sin = st["cos"][st["positions"]].unsqueeze(1), st["sin"][st["positions"]].unsqueeze(1)
        t = x[:, :H + Hk].float()
        turned = torch.cat((-t[..., hd // 2:], t[..., :hd // 2]), -1)
        t = (t * cos + turned * sin).to(x.dtype)
        q = t[:, :H].contiguous()
        at, off = st["slots"] // page, st["slots"] % page
        kv = []
        for i, (rows, pages) in enumerate(((t[:, H:], kp), (x[:, H + Hk:], vp))):
            n, step, zero = _to_4bit(rows)
            pages[at, :, off] = n[..., 0::2] | n[..., 1::2] << 4
            scales[at, :, off, :, 2 * i] = step.bfloat16()
            scales[at, :, off, :, 2 * i + 1] = zero.bfloat16()
            kv.append(_from_4bit(n, step, zero).to(x.dtype))
        k, v = kv
    # k and v are what the filed numbers stand for
    return {"q": q, "k": k, "v": v, "k_pages": kp, "v_pages": vp, "scales": scales}


def _rows(st, b, n, dtype):
    """Keys and values (Hk, n, hd) of sequence b as the cache holds them."""
    page = st["case"]["page"]
    ids = st["table"][b, :-(-n // page)].long()
    out = []
    for i, pages in enumerate((st["k_pages"], st["v_pages"])):
        raw = pages[ids].transpose(0, 1).flatten(1, 2)[:, :n]
        s = st["scales"][ids].transpose(0, 1).flatten(1, 2)[:, :n].to(dtype)
        num = torch.stack((raw & 15, raw >> 4), -1).flatten(-2).to(dtype).unflatten(-1, (-1, GROUP))
        out.append((num * s[..., 2 * i, None] + s[..., 2 * i + 1, None]).flatten(-2))
    return out


def _run_decode(st):
    case = st["case"]
    q = st["q"]
    if own:
        from naylis_b200 import attention
        return attention.decode_attention_int4(q, st["k_pages"], st["v_pages"], st["scales"], st["table"],
                                               st["seq_lens"], new_lens=st.get("new_lens"), scale=st["scale"],
                                               max_len=case["longest"])
    Hk, G, hd = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"]
    out = torch.zeros_like(q)
    for b, n in enumerate(st["lens"]):
        m = st["new"][b]
        k, v = _rows(st, b, n, torch.float32)
        # a head's new tokens, one group of query heads after another: (Hk, m G, hd)
        qs = q[b, :m].float().view(m, Hk, G, hd).transpose(0, 1).reshape(Hk, m * G, hd)
        s = torch.matmul(qs, k.transpose(1, 2)) * st["scale"]
        if m > 1:
            sees = n - m + 1 + torch.arange(m, device=q.device).repeat_interleave(G)
            s.masked_fill_(torch.arange(n, device=q.device)[None, :] >= sees[:, None], float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[b, :m] = o.view(Hk, m, G, hd).transpose(0, 1).reshape(m, Hk * G, hd).to(q.dtype)
    return out


def _run_verify(st):
    case, logits, drafts, u = st["case"], st["logits"], st["drafts"], st["uniforms"]
    T = case["temperature"]
    if own:
        from naylis_b200 import scoring
        r = scoring.verify_drafts(logits, drafts, u, draft_logits=st["draft_logits"], temperature=T,
                                  draft_lens=st["draft_lens"])
        return {"tokens": r.tokens, "accepted": r.accepted}
    B, K = drafts.shape
    V = logits.shape[2]
    tokens = torch.empty(B, K + 1, dtype=torch.int64, device=DEV)
    accepted = torch.empty(B, dtype=torch.int64, device=DEV)
    step = max(1, (1 << 26) // ((K + 1) * V))
    for a in range(0, B, step):
        b = min(B, a + step)
        lens, x = st["draft_lens"][a:b, None].long(), drafts[a:b]
        col = torch.arange(K + 1, device=DEV)
        if case["mode"] == "greedy":
            y = logits[a:b].float()
            at = torch.where(y == y.amax(-1, keepdim=True), torch.arange(V, device=DEV), V).amin(-1)
            ok = x == at[:, :K]
        else:
            # in 64 bits: a sum over the vocabulary decides between neighbouring tokens
            def soft(z):
                z = z.double()
                e = torch.exp((z - z.amax(-1, keepdim=True)) / T)
                return e / e.sum(-1, keepdim=True)

            p = soft(logits[a:b])
            px = p[:, :K].gather(2, x[..., None])[..., 0]
            if st["draft_logits"] is not None:
                q = soft(st["draft_logits"][a:b])
                qx = q.gather(2, x[..., None])[..., 0]
            else:
                q = torch.zeros_like(p[:, :K]).scatter_(2, x[..., None], 1.0)
                qx = torch.ones_like(px)
            ok = px > u[a:b, :K].double() * qx
        ok = ok & (col[:K] < lens)
        n = torch.cumprod(ok.long(), 1).sum(1)
        if case["mode"] == "greedy":
            nxt = at.gather(1, n[:, None])[:, 0]
        else:
            row = torch.arange(b - a, device=DEV)
            r = p[row, n]
            cut = n < lens[:, 0]
            left = (r - q[row, n.clamp_max(K - 1)]).clamp_min(0.0)
            r = torch.where((cut & (left.sum(1) > 0))[:, None], left, r)
            c = torch.cumsum(r, 1)
            thr = u[a:b, K].double() * c[:, -1]
            nxt = torch.searchsorted(c, thr[:, None], right=True)[:, 0]
            last = torch.where(r > 0, torch.arange(V, device=DEV), 0).amax(1)
            nxt = torch.minimum(nxt, last)
        got = torch.cat((x, x[:, :1]), 1)
        got = torch.where(col == n[:, None], nxt[:, None], got)
        tokens[a:b] = torch.where(col <= n[:, None], got, -1)
        accepted[a:b] = n
    return {"tokens": tokens, "accepted": accepted}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "verify":
        B, K, V = case["seqs"], case["drafts"], case["vocab"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        n = B * V * (K + 1 + (K if case["mode"] == "sampled" else 0))
        return {"bytes": n * size + B * (8 * K + 4 * (K + 1) + 4 + 8 * (K + 2)), "flops": 4 * n}
    H, Hk, hd, lens = case["heads"], case["kv_heads"], case["head_dim"], lengths(case)
    row = hd // 2 + 4 * (hd // GROUP)           # of a key or a value, with its scale and zero
    T = sum(lens)
    if op == "decode":
        new = new_tokens(case)
        pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, new))
        return {"bytes": 2 * row * T * Hk + 4 * hd * H * len(lens) * case["new"] +
                4 * sum(-(-n // case["page"]) for n in lens) + 8 * len(lens), "flops": 4 * hd * H * pairs}
    most = max(lens) + case["past"]
    return {"bytes": 2 * hd * T * (H + 2 * Hk) + 2 * hd * T * (H + 2 * Hk) + 2 * row * T * Hk + 16 * T +
            8 * hd * min(most, T), "flops": T * hd * (3 * (H + Hk) + 10 * Hk)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "verify": _exact_verify}[case["op"]](st)


def _exact_append(st):
    case = st["case"]
    H, Hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    x = st["qkv"].view(-1, H + 2 * Hk, hd)
    c, s = (st[t][st["positions"]].double()[:, None, :hd // 2] for t in ("cos", "sin"))
    lo, hi = x[:, :H + Hk, :hd // 2].double(), x[:, :H + Hk, hd // 2:].double()
    turned = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
    # what 4 bits keep of the values, whose inputs are exact; a rotated key's number hangs on its rounding
    v = x[:, H + Hk:].double().reshape(-1, GROUP)
    least, most = v.min(1)[0][:, None], v.max(1)[0][:, None]
    step = ((most - least) / 15).float().bfloat16().double()
    v = least + step * torch.clamp(torch.round((v - least) / step), 0, 15)
    return {"q": turned[:, :H].contiguous(), "k": None, "v": v.reshape(-1, Hk, hd), "k_pages": None, "v_pages": None,
            "scales": None}


def _exact_decode(st):
    case = st["case"]
    Hk, G, hd, page = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["lens"]):
        t = torch.arange(n, device=DEV)
        ids, off = st["table"][b].long()[t // page], t % page
        m = st["new"][b]
        for h in range(Hk):
            kv = []
            for i, pages in enumerate((st["k_pages"], st["v_pages"])):
                raw = pages[ids, h, off].long()
                num = torch.empty(n, hd, dtype=torch.float64, device=DEV)
                num[:, 0::2], num[:, 1::2] = (raw % 16).double(), (raw // 16).double()
                sz = st["scales"][ids, h, off].double().repeat_interleave(GROUP, 1)
                kv.append(sz[..., 2 * i + 1] + num * sz[..., 2 * i])
            for j in range(m):
                e = n - m + 1 + j
                w = torch.softmax(st["q"][b, j, h * G:(h + 1) * G].double() @ kv[0][:e].T * hd ** -0.5, -1)
                out[b, j, h * G:(h + 1) * G] = w @ kv[1][:e]
    return out


def _exact_verify(st):
    case, T = st["case"], st["case"]["temperature"]
    B, K = st["drafts"].shape
    drafts, lens = st["drafts"].tolist(), st["draft_lens"].tolist()
    u = None if st["uniforms"] is None else st["uniforms"].double().tolist()
    tokens, accepted = torch.full((B, K + 1), -1, dtype=torch.int64), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        row = []
        while True:
            j = len(row)
            x = st["logits"][b, j].double()
            if T == 0:
                best = int((x == x.max()).nonzero()[0])
                if j < lens[b] and drafts[b][j] == best:
                    row.append(best)
                    continue
                row.append(best)
                break
            p = torch.softmax(x / T, -1)
            if j == lens[b]:
                r = p
            else:
                d = drafts[b][j]
                q = torch.zeros_like(p)
                q[d] = 1.0
                if st["draft_logits"] is not None:
                    q = torch.softmax(st["draft_logits"][b, j].double() / T, -1)
                if u[b][j] * float(q[d]) < float(p[d]):
                    row.append(d)
                    continue
                r = torch.relu(p - q)
                r = p if float(r.sum()) == 0.0 else r
            c = r.cumsum(0)
            row.append(min(int((c <= u[b][K] * c[-1]).sum()), int(r.nonzero()[-1])))
            break
        tokens[b, :len(row)] = torch.tensor(row)
        accepted[b] = len(row) - 1
    return {"tokens": tokens.to(DEV), "accepted": accepted.to(DEV)}
