"""The serving and scoring operators as a user calls them, next to their plain forms.

Four operators carry a request through the decoder: ``rope_append`` rotates a
projection's heads and files keys and values into the paged cache,
``prompt_attention`` attends over packed prompts, ``decode_attention`` attends
one new token of each sequence over its pages, ``token_logprobs`` scores the LM
head's logits (log probabilities, entropy, top alternatives, and the gradient
that a policy update needs).

A case is a dict of plain values. Sequence lengths of a batch are spread from
its ``longest`` down by ``lengths`` below, so a case names them by three numbers.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one short chat turn on an idle server: latency
        {"name": "prompt-one-128", "op": "prompt", "seqs": 1, "longest": 128, "spread": 1.0, "past": 0,
         "heads": 16, "kv_heads": 16, "head_dim": 64},
        # the decoder's own geometry: 8 sequences of 2048, 16 heads of 64, one head of keys each
        {"name": "prompt-8x2048", "op": "prompt", "seqs": 8, "longest": 2048, "spread": 1.0, "past": 0,
         "heads": 16, "kv_heads": 16, "head_dim": 64},
        # a busy server's packed prompts, from 1 token to 4099, grouped heads of 128
        {"name": "prompt-packed-24", "op": "prompt", "seqs": 24, "longest": 4099, "spread": 4099.0, "past": 0,
         "heads": 16, "kv_heads": 4, "head_dim": 128},
        # one long document
        {"name": "prompt-16384", "op": "prompt", "seqs": 1, "longest": 16384, "spread": 1.0, "past": 0,
         "heads": 16, "kv_heads": 4, "head_dim": 128},
        # one user's next token: latency
        {"name": "decode-one-577", "op": "decode", "seqs": 1, "longest": 577, "spread": 1.0,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16},
        # a batch of conversations of very different lengths, the decoder's own heads
        {"name": "decode-48-ragged", "op": "decode", "seqs": 48, "longest": 4096, "spread": 64.0,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 32},
        # a few long documents, grouped heads
        {"name": "decode-4x131072", "op": "decode", "seqs": 4, "longest": 131072, "spread": 1.5,
         "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 64},
        # one decode step's keys and values of 64 sequences
        {"name": "append-step-64", "op": "append", "seqs": 64, "longest": 1, "spread": 1.0, "past": 1500,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16},
        # a prefill's 16 thousand tokens
        {"name": "append-prompt-8x2048", "op": "append", "seqs": 8, "longest": 2048, "spread": 1.0, "past": 0,
         "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 64},
        # the sampled tokens of one decode step, with 8 alternatives
        {"name": "logprobs-step-16", "op": "logprobs", "rows": 16, "vocab": 32000, "dtype": "bfloat16", "top": 8,
         "temperature": 1.0, "grad": False},
        # a policy update over 8 sequences of 2048: log probabilities, entropy and the logits' gradient
        {"name": "logprobs-train-8x2047", "op": "logprobs", "rows": 16376, "vocab": 32000, "dtype": "bfloat16",
         "top": 0, "temperature": 1.0, "grad": True},
        # evaluation in fp32 with an odd vocabulary, 20 alternatives and their gradient
        {"name": "logprobs-odd-fp32", "op": "logprobs", "rows": 1021, "vocab": 32003, "dtype": "float32", "top": 20,
         "temperature": 0.7, "grad": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "decode", "append", "logprobs"])
    if op == "logprobs":
        c = {"op": op, "vocab": _log_int(rng, 2, 65000), "dtype": rng.choice(["bfloat16", "float32"]),
             "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]), "grad": rng.random() < 0.5}
        c["rows"] = _log_int(rng, 1, min(16376, 16376 * 32000 // (2 * c["vocab"])))
        c["top"] = min(c["vocab"], rng.choice([0, 1, 5, 8, 20, 32]))
        return c
    c = {"op": op, "head_dim": rng.choice([64, 128]), "kv_heads": rng.choice([1, 2, 4, 8, 16])}
    c["heads"] = c["kv_heads"] * rng.choice([g for g in (1, 2, 4, 8, 16) if g * c["kv_heads"] <= 32])
    c["seqs"] = _log_int(rng, 1, 64)
    c["spread"] = rng.choice([1.0, 1.5, 8.0, 100.0])
    if op == "prompt":
        c["past"] = rng.choice([0, 0, 0, _log_int(rng, 1, 4096)])
        most = 16384 ** 2 * 16 * 128 // 3
        c["longest"] = _log_int(rng, 1, 16384)
        while c["seqs"] > 1 and c["seqs"] * c["longest"] * (c["longest"] + 2 * c["past"]) * c["heads"] * c["head_dim"] > most:
            c["seqs"] -= 1
        while c["longest"] > 1 and c["longest"] * (c["longest"] + 2 * c["past"]) * c["heads"] * c["head_dim"] > most:
            c["longest"] = c["longest"] * 7 // 8
        return c
    c["page"] = rng.choice([8, 16, 32, 64, 128])
    if op == "append":
        c["past"] = rng.choice([0, _log_int(rng, 1, 4096)])
        c["longest"] = _log_int(rng, 1, max(1, min(8192, 8 * 2048 * 24 * 128 // (
            c["seqs"] * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]))))
        return c
    c["longest"] = _log_int(rng, 1, min(131072, 4 * 131072 * 4 * 128 // (2 * c["seqs"] * c["kv_heads"] * c["head_dim"])))
    return c


def lengths(case):
    """The batch's lengths: from `longest` down to longest / spread, evenly in the logarithm, in a mixed order."""
    n, hi = case["seqs"], case["longest"]
    lo = max(1.0, hi / case["spread"])
    got = [hi if n == 1 else max(1, int(round(hi * (lo / hi) ** (i / (n - 1))))) for i in range(n)]
    return [int(got[i]) for i in np.random.RandomState(7).permutation(n)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 26):      # bounded fp32 temporaries
        n = min(1 << 26, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=DEV) * scale
    return out


def _pages(case, lens, seed):
    """A cache after long use: every sequence's pages scattered over the pool. -> (pages, table)"""
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


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "logprobs":
        R, V = case["rows"], case["vocab"]
        dt = getattr(torch, case["dtype"])
        # an LM head's logits: a few units wide, with some clear favourites
        logits = _randn(g, R, V, scale=2.0, dtype=dt)
        fav = torch.randint(0, V, (R, 4), generator=g, device=DEV)
        logits.scatter_(1, fav, (6.0 + 3.0 * torch.rand(R, 4, generator=g, device=DEV)).to(dt))
        targets = torch.where(torch.rand(R, generator=g, device=DEV) < 0.5, fav[:, 0],
                              torch.randint(0, V, (R,), generator=g, device=DEV))
        if case["grad"]:
            targets[torch.rand(R, generator=g, device=DEV) < 0.1] = -100      # prompt positions
        st = {"case": case, "logits": logits, "targets": targets}
        if case["grad"]:
            st["g_logprob"] = torch.randn(R, generator=g, device=DEV)
            st["g_entropy"] = -0.01 * torch.ones(R, device=DEV)
            if case["top"]:
                st["g_top"] = torch.randn(R, case["top"], generator=g, device=DEV)
            if own:
                logits.requires_grad_(True)
        return st
    H, Hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lens = lengths(case)
    st = {"case": case, "lens": lens, "scale": hd ** -0.5}
    if op == "prompt":
        T, past = sum(lens), case["past"]
        Tk = T + past * len(lens)
        st["q"] = _randn(g, T, H, hd, scale=2.0)
        st["k"] = _randn(g, Tk, Hk, hd)
        # the values stay where the fused projection wrote them: a strided view
        st["v"] = _randn(g, Tk, 2 * Hk, hd)[:, Hk:]
        if own:
            from naylis_b200 import attention
            st["plan"] = attention.PromptPlan(lens, [n + past for n in lens] if past else None, device=DEV)
        return st
    if op == "decode":
        total, table = _pages(case, lens, seed)
        st["q"] = _randn(g, len(lens), H, hd, scale=2.0)
        st["k_pages"] = _randn(g, total, Hk, case["page"], hd)
        st["v_pages"] = _randn(g, total, Hk, case["page"], hd)
        st["table"] = table.to(DEV)
        st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        return st
    past = case["past"]
    full = [n + past for n in lens]
    total, table = _pages(case, full, seed)
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
    st["k_pages"] = _randn(g, total, Hk, case["page"], hd)
    st["v_pages"] = _randn(g, total, Hk, case["page"], hd)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    return {"prompt": _run_prompt, "decode": _run_decode, "append": _run_append,
            "logprobs": _run_logprobs}[state["case"]["op"]](state)


def _run_prompt(st):
    if own:
        from naylis_b200 import attention
        return attention.prompt_attention(st["q"], st["k"], st["v"], st["plan"], scale=st["scale"])
    q, k, v, past = st["q"], st["k"], st["v"], st["case"]["past"]
    H, Hk = q.shape[1], k.shape[1]
    out = torch.empty_like(q)
    o, ok = 0, 0
    for n in st["lens"]:
        m = n + past
        step = max(1, min(Hk, (1 << 31) // (n * m * (H // Hk))))          # key heads at a time
        for h in range(0, Hk, step):
            h1 = min(Hk, h + step)
            G = H // Hk
            qs = q[o:o + n, h * G:h1 * G].float().view(n, h1 - h, G, -1).permute(1, 2, 0, 3)
            ks = k[ok:ok + m, h:h1].float().permute(1, 2, 0).unsqueeze(1)
            vs = v[ok:ok + m, h:h1].float().permute(1, 0, 2).unsqueeze(1)
            s = torch.matmul(qs, ks) * st["scale"]
            rows = torch.arange(n, device=q.device)[:, None] + past
            s.masked_fill_(torch.arange(m, device=q.device)[None, :] > rows, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            y = torch.matmul(p, vs) / p.sum(-1, keepdim=True)
            out[o:o + n, h * G:h1 * G] = y.permute(2, 0, 1, 3).reshape(n, (h1 - h) * G, -1).to(q.dtype)
            del s, p, y
        o, ok = o + n, ok + m
    return out


def _run_decode(st):
    case = st["case"]
    if own:
        from naylis_b200 import attention
        return attention.decode_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seq_lens"],
                                          scale=st["scale"], max_len=case["longest"])
    q, page = st["q"], case["page"]
    Hk, G, hd = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"]
    out = torch.empty_like(q)
    for b, n in enumerate(st["lens"]):
        ids = st["table"][b, :-(-n // page)].long()
        k = st["k_pages"][ids].permute(1, 0, 2, 3).reshape(Hk, -1, hd)[:, :n].float()
        v = st["v_pages"][ids].permute(1, 0, 2, 3).reshape(Hk, -1, hd)[:, :n].float()
        s = torch.matmul(q[b].float().view(Hk, G, hd), k.transpose(1, 2)) * st["scale"]
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[b] = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(Hk * G, hd).to(q.dtype)
    return out


def _run_append(st):
    case = st["case"]
    H, Hk, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    prompt = case["longest"] > 1                # a prefill also wants the keys side by side
    if own:
        from naylis_b200 import attention
        q, k = attention.rope_append(st["qkv"], st["cos"], st["sin"], st["positions"], st["k_pages"], st["v_pages"],
                                     st["slots"], n_heads=H, want_k=prompt)
    else:
        x = st["qkv"].view(-1, H + 2 * Hk, hd)
        cos, sin = st["cos"][st["positions"]].unsqueeze(1), st["sin"][st["positions"]].unsqueeze(1)

        def rotate(t):
            t = t.float()
            turned = torch.cat((-t[..., hd // 2:], t[..., :hd // 2]), -1)
            return (t * cos + turned * sin).to(x.dtype)

        q, k = rotate(x[:, :H]), rotate(x[:, H:H + Hk])
        at, off = st["slots"] // page, st["slots"] % page
        st["k_pages"][at, :, off] = k
        st["v_pages"][at, :, off] = x[:, H + Hk:]
    return {"q": q, **({"k": k} if prompt else {}), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _ranked(x, top):
    """The `top` greatest of each row of fp32 x, ties to the lowest index."""
    V = x.shape[1]
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    key = order * (1 << 32) + (V - 1 - torch.arange(V, device=x.device))
    return torch.topk(key, top, dim=-1)[1]


def _run_logprobs(st):
    case, logits, targets = st["case"], st["logits"], st["targets"]
    top, grad = case["top"], case["grad"]
    if own:
        from naylis_b200 import scoring
        r = scoring.token_logprobs(logits, targets, top_k=top, temperature=case["temperature"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if top:
            out.update(top_logprob=r.top_logprob, top_idx=r.top_idx)
        if grad:
            ys = [r.logprob, r.entropy] + ([r.top_logprob] if top else [])
            gs = [st["g_logprob"], st["g_entropy"]] + ([st["g_top"]] if top else [])
            out["dlogits"], = torch.autograd.grad(ys, logits, gs)
        return out
    R, V = logits.shape
    out = {"logprob": torch.empty(R, device=DEV), "entropy": torch.empty(R, device=DEV)}
    if top:
        out["top_logprob"] = torch.empty(R, top, device=DEV)
        out["top_idx"] = torch.empty(R, top, dtype=torch.int64, device=DEV)
    if grad:
        out["dlogits"] = torch.empty_like(logits)
    step = max(1, (1 << 28) // V)
    for a in range(0, R, step):
        b = min(R, a + step)
        x = logits[a:b].float()
        y = x / case["temperature"]
        y = y - y.amax(-1, keepdim=True)
        e = torch.exp(y)
        z = e.sum(-1, keepdim=True)
        lp = y - torch.log(z)
        p = e / z
        live = targets[a:b] != -100
        t = targets[a:b].clamp_min(0)[:, None]
        out["logprob"][a:b] = torch.where(live, lp.gather(1, t)[:, 0], 0.0)
        h = -(p * lp).sum(-1)
        out["entropy"][a:b] = h
        if top:
            idx = _ranked(x, top)
            out["top_idx"][a:b] = idx
            out["top_logprob"][a:b] = lp.gather(1, idx)
        if grad:
            gl = torch.where(live, st["g_logprob"][a:b], 0.0)[:, None]
            d = -(p * (lp + h[:, None])) * st["g_entropy"][a:b, None] - p * gl
            d.scatter_add_(1, t, gl)
            if top:
                gt = st["g_top"][a:b]
                d -= p * gt.sum(-1, keepdim=True)
                d.scatter_add_(1, idx, gt)
            out["dlogits"][a:b] = (d / case["temperature"]).to(logits.dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "logprobs":
        R, V, top = case["rows"], case["vocab"], case["top"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        n = R * V
        return {"bytes": n * size * (2 if case["grad"] else 1) + R * (16 + 12 * top),
                "flops": n * (6 + (6 if case["grad"] else 0))}
    H, Hk, hd, lens = case["heads"], case["kv_heads"], case["head_dim"], lengths(case)
    T = sum(lens)
    if op == "prompt":
        past = case["past"]
        Tk = T + past * len(lens)
        pairs = sum(n * past + n * (n + 1) // 2 for n in lens)
        return {"bytes": 2 * hd * (2 * T * H + 2 * Tk * Hk), "flops": 4 * hd * H * pairs}
    if op == "decode":
        return {"bytes": 2 * hd * (2 * T * Hk + 2 * len(lens) * H) + 4 * sum(-(-n // case["page"]) for n in lens),
                "flops": 4 * hd * H * T}
    most = max(lens) + case["past"]
    k_side = Hk if case["longest"] > 1 else 0
    return {"bytes": 2 * hd * T * (2 * (H + 2 * Hk) + k_side) + 16 * T + 8 * hd * min(most, T),
            "flops": 3 * hd * T * (H + Hk)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        return _exact_logprobs(st)
    H, Hk, hd, lens = case["heads"], case["kv_heads"], case["head_dim"], st["lens"]
    G = H // Hk
    if op == "append":
        x = st["qkv"].double().view(-1, H + 2 * Hk, hd)
        c, s = (st[t][st["positions"]].double()[:, None, :hd // 2] for t in ("cos", "sin"))
        lo, hi = x[:, :H + Hk, :hd // 2], x[:, :H + Hk, hd // 2:]
        turned = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        page = case["page"]
        for t0 in range(0, x.shape[0], 4096):
            sl = st["slots"][t0:t0 + 4096]
            kp[sl // page, :, sl % page] = turned[t0:t0 + 4096, H:]
            vp[sl // page, :, sl % page] = x[t0:t0 + 4096, H + Hk:]
        out = {"q": turned[:, :H].contiguous(), "k_pages": kp, "v_pages": vp}
        if case["longest"] > 1:
            out["k"] = turned[:, H:].contiguous()
        return out
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    if op == "decode":
        page = case["page"]
        for b, n in enumerate(lens):
            t = torch.arange(n, device=DEV)
            ids, off = st["table"][b].long()[t // page], t % page
            for h in range(Hk):
                k, v = st["k_pages"][ids, h, off].double(), st["v_pages"][ids, h, off].double()
                w = torch.softmax(st["q"][b, h * G:(h + 1) * G].double() @ k.T * hd ** -0.5, -1)
                out[b, h * G:(h + 1) * G] = w @ v
        return out
    past, o, ok = case["past"], 0, 0
    for n in lens:
        m = n + past
        for h in range(H):
            k, v = st["k"][ok:ok + m, h // G].double(), st["v"][ok:ok + m, h // G].double()
            for r in range(0, n, 4096):
                r1 = min(n, r + 4096)
                e = past + r1                       # no row of this piece sees a key at or after e
                s = st["q"][o + r:o + r1, h].double() @ k[:e].T * hd ** -0.5
                seen = torch.ones(r1 - r, e, dtype=torch.bool, device=DEV).tril(past + r)
                out[o + r:o + r1, h] = torch.softmax(torch.where(seen, s, -math.inf), -1) @ v[:e]
        o, ok = o + n, ok + m
    return out


def _exact_logprobs(st):
    case = st["case"]
    R, V, top, T = case["rows"], case["vocab"], case["top"], case["temperature"]
    parts = {"logprob": [], "entropy": [], "top_logprob": [], "dlogits": []}
    for a in range(0, R, 1024):
        b = min(R, a + 1024)
        x = st["logits"].detach()[a:b].double()
        lp = torch.log_softmax(x / T, -1)
        p = lp.exp()
        h = -(p * lp).sum(-1)
        live = st["targets"][a:b] >= 0
        t = torch.where(live, st["targets"][a:b], 0)[:, None]
        parts["logprob"].append(lp.gather(1, t)[:, 0] * live)
        parts["entropy"].append(h)
        best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top] if top else None
        if top:
            parts["top_logprob"].append(lp.gather(1, best))
        if case["grad"]:
            pick = torch.zeros_like(p).scatter_add_(1, t, (st["g_logprob"][a:b].double() * live)[:, None])
            if top:
                pick.scatter_add_(1, best, st["g_top"][a:b].double())
            d = pick - p * pick.sum(-1, keepdim=True)
            d -= st["g_entropy"][a:b, None].double() * p * (lp + h[:, None])
            parts["dlogits"].append(d / T)
    out = {k: torch.cat(v) for k, v in parts.items() if v}
    if top:
        out["top_idx"] = None
    return out
