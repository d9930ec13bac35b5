"""GPU tests of the serving operators (naylis_b200/attention.py) against their
definitions in 64 bits on the same bf16 inputs.

Tolerance of attention, per element, from the roundings the kernels may take: the
output is rounded to bf16 (8 significant bits, half an ulp: 2^-8 of |o|), the
weights may be rounded to bf16 before they meet the values (2^-8 of
A = sum_j p_j |v_j|, which bounds |o|), the exponential is within 2^-13 (of A), and
fp32 sums are far below. So |out - exact| <= (2^-7 + 2^-12) A, held for every
element; 2^-40 covers A = 0.
rope_append is exact: two fp32 products and a sum rounded once, as torch's ops.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TOL = 2.0 ** -7 + 2.0 ** -12


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(DEV)


def _attend(q, k, v, visible, scale):
    """q (n, H, hd), k / v (m, Hk, hd), visible (n, m) bool -> (out, A) in 64 bits;
    hidden values are left out, so what they hold does not matter."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    out, A = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(n):
        j = visible[i].nonzero()[:, 0]
        if len(j):
            p = torch.softmax(torch.einsum("hd,jhd->hj", q[i], k[j]) * scale, -1)
            out[i] = torch.einsum("hj,jhd->hd", p, v[j])
            A[i] = torch.einsum("hj,jhd->hd", p, v[j].abs())
    return out, A


def _close(got, out, A):
    err = (got.double() - out).abs()
    assert bool(torch.isfinite(got).all())
    worst = float((err - TOL * A).max())
    assert worst <= 2.0 ** -40, (worst, float(err.max()))


def _prompt_exact(q, k, v, q_lens, k_lens, scale):
    outs, As = [], []
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        vis = torch.arange(m, device=DEV)[None, :] <= torch.arange(n, device=DEV)[:, None] + (m - n)
        o, A = _attend(q[a:a + n], k[b:b + m], v[b:b + m], vis, scale)
        outs.append(o)
        As.append(A)
        a, b = a + n, b + m
    return torch.cat(outs), torch.cat(As)


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("hd,H,Hk", [(64, 2, 2), (128, 4, 1), (64, 6, 2), (128, 3, 3)])
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1], None), ([127], None), ([128], None), ([129, 1, 2], None), ([256], None), ([257, 31], None),
    ([5, 300, 1, 64, 0, 130], None), ([513], None),
    ([1, 7, 130], [300, 7, 258]),            # a cached prefix
    ([64, 3], [10, 0]),                      # rows before the first key, a sequence without keys
    ([128, 200], [129, 455]),
])
def test_prompt_attention(hd, H, Hk, q_lens, k_lens):
    from naylis_b200 import attention
    ks = k_lens or q_lens
    q = _rand(1, sum(q_lens), H, hd, scale=2.0)
    k, v = _rand(2, sum(ks), Hk, hd), _rand(3, sum(ks), Hk, hd)
    plan = attention.PromptPlan(q_lens, k_lens, device=DEV)
    out = attention.prompt_attention(q, k, v, plan)
    plan.check()
    _close(out, *_prompt_exact(q, k, v, q_lens, ks, hd ** -0.5))
    again = attention.prompt_attention(q, k, v, plan)
    assert torch.equal(out, again)


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attention_takes_the_projection_as_it_is(hd):
    """q, k and v as views of one fused projection, odd sizes, on a stream of its own."""
    from naylis_b200 import attention
    lens, H, Hk = [77, 300, 1], 4, 2
    qkv = _rand(4, sum(lens), H + 2 * Hk, hd)
    plan = attention.PromptPlan(lens, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = attention.prompt_attention(qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], plan, scale=0.2)
    s.synchronize()
    q, k, v = (t.contiguous() for t in (qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]))
    _close(out, *_prompt_exact(q, k, v, lens, lens, 0.2))
    # heads in another order than memory's: the operator copies
    flipped = attention.prompt_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, plan, scale=0.2)
    assert torch.equal(out, flipped)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_attention_hidden_values_stay_hidden(hd, bad):
    """A value (or key) that the mask hides from a row does not reach it, whatever it
    holds; one that a row sees does. Sequence 1 holds the bad value at key 140."""
    from naylis_b200 import attention
    lens, H, Hk, at = [100, 200, 90], 4, 2, 140
    q = _rand(5, sum(lens), H, hd)
    k, v = _rand(6, sum(lens), Hk, hd), _rand(7, sum(lens), Hk, hd)
    plan = attention.PromptPlan(lens, device=DEV)
    want, A = _prompt_exact(q, k, v, lens, lens, hd ** -0.5)
    row = lens[0] + at
    v2 = v.clone()
    v2[row, 1, 5] = bad
    out = attention.prompt_attention(q, k, v2, plan)
    seen = torch.zeros(sum(lens), H, hd, dtype=torch.bool, device=DEV)
    seen[row:lens[0] + lens[1], 2:, 5] = True
    _close(out[~seen], want[~seen], A[~seen])
    hit = out[seen].float()
    assert bool((torch.isnan(hit) if math.isnan(bad) else hit == bad).all())
    k2 = k.clone()
    k2[row, 1, 5] = float("nan")
    out = attention.prompt_attention(q, k2, v, plan)
    seen = torch.zeros(sum(lens), H, hd, dtype=torch.bool, device=DEV)
    seen[row:lens[0] + lens[1], 2:] = True
    _close(out[~seen], want[~seen], A[~seen])
    assert bool(torch.isnan(out[seen].float()).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attention_wide_scores(hd):
    """Scores hundreds of units apart, rising along the row so that the running
    maximum moves at every tile, and falling."""
    from naylis_b200 import attention
    n, H = 700, 2
    q = torch.ones(n, H, hd, device=DEV).to(torch.bfloat16)
    ramp = torch.linspace(-300, 300, n, device=DEV)
    k = torch.zeros(n, H, hd, device=DEV)
    k[:, 0, 0], k[:, 1, 0] = ramp, -ramp
    k = k.to(torch.bfloat16)
    v = _rand(8, n, H, hd)
    plan = attention.PromptPlan([n], device=DEV)
    out = attention.prompt_attention(q, k, v, plan, scale=1.0)
    _close(out, *_prompt_exact(q, k, v, [n], [n], 1.0))


@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (64, 4, 2), (128, 4, 1), (128, 3, 3)])
@pytest.mark.parametrize("n,seqs,past", [(100, 400, 0), (300, 120, 0), (129, 250, 0), (40, 500, 90), (700, 40, 0)])
def test_prompt_attention_many_tiles(hd, H, Hk, n, seqs, past):
    """Several work items for every CTA, down to single key tiles: equal sequences,
    compared as one batch."""
    from naylis_b200 import attention
    m = n + past
    q = _rand(90, seqs * n, H, hd, scale=2.0)
    k, v = _rand(91, seqs * m, Hk, hd), _rand(92, seqs * m, Hk, hd)
    plan = attention.PromptPlan([n] * seqs, [m] * seqs, device=DEV)
    out = attention.prompt_attention(q, k, v, plan)
    for _ in range(3):
        assert torch.equal(out, attention.prompt_attention(q, k, v, plan))
    plan.check()
    seen = torch.ones(n, m, dtype=torch.bool, device=DEV).tril(past)
    for b in range(0, seqs, 50):
        e = min(seqs, b + 50)
        qb = q[b * n:e * n].double().view(e - b, n, H, hd).transpose(1, 2)
        kb, vb = (t[b * m:e * m].double().view(e - b, m, Hk, hd).transpose(1, 2).repeat_interleave(H // Hk, 1)
                  for t in (k, v))
        s = (qb @ kb.transpose(2, 3) * hd ** -0.5).masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1)
        flat = lambda t: t.transpose(1, 2).reshape(-1, H, hd)
        _close(out[b * n:e * n], flat(p @ vb), flat(p @ vb.abs()))


def test_prompt_attention_refuses():
    from naylis_b200 import attention
    plan = attention.PromptPlan([4, 5], device=DEV)
    q, k = _rand(1, 9, 4, 64), _rand(2, 9, 2, 64)
    ok = attention.prompt_attention(q, k, k, plan)
    assert ok.shape == (9, 4, 64)
    empty = attention.PromptPlan([], device=DEV)
    assert attention.prompt_attention(q[:0], k[:0], k[:0], empty).shape == (0, 4, 64)
    for args in [(q.float(), k, k, plan), (q, k.half(), k, plan), (q[:8], k, k, plan), (q, k[:8], k[:8], plan),
                 (q, k, _rand(3, 9, 4, 64), plan), (_rand(1, 9, 3, 64), k, k, plan), (q[0], k, k, plan),
                 (_rand(1, 9, 4, 32), _rand(2, 9, 2, 32), _rand(2, 9, 2, 32), plan), (q.cpu(), k, k, plan)]:
        with pytest.raises(RuntimeError):
            attention.prompt_attention(*args)
    with pytest.raises(RuntimeError):
        attention.prompt_attention(q.clone().requires_grad_(True), k, k, plan)
    for scale in (float("nan"), 0.0, -0.1):
        with pytest.raises(RuntimeError):
            attention.prompt_attention(q, k, k, plan, scale=scale)
    for ql, kl in [([3, -1], None), ([3], [1, 2]), ([1], [-2]), ([1 << 31], None)]:
        with pytest.raises(RuntimeError):
            attention.PromptPlan(ql, kl, device=DEV)


# ------------------------------------------------------------------ decode
def _cache(seed, lens, Hk, page, hd, extra=2, fill=None):
    """Scattered pages holding k, v of each sequence; what no sequence owns is `fill`."""
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + extra
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    kp, vp = _rand(seed + 1, total, Hk, page, hd), _rand(seed + 2, total, Hk, page, hd)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    ks, vs = [], []
    for b, n in enumerate(lens):
        ids = [perm.pop() for _ in range(need[b])]
        table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        if fill is not None and n > 0 and n % page:
            kp[ids[-1], :, n % page:] = fill
            vp[ids[-1], :, n % page:] = fill
        flat = lambda t: (t[ids].transpose(1, 2).reshape(-1, Hk, hd)[:max(n, 0)] if ids
                          else t.new_zeros(0, Hk, hd))
        ks.append(flat(kp))
        vs.append(flat(vp))
    if fill is not None:
        for i in perm:
            kp[i] = fill
            vp[i] = fill
    return kp, vp, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), ks, vs


def _decode_exact(q, ks, vs, scale):
    pairs = [_attend(q[b:b + 1], k, v, torch.ones(1, k.shape[0], dtype=torch.bool, device=DEV), scale)
             for b, (k, v) in enumerate(zip(ks, vs))]
    return torch.cat([p[0] for p in pairs]), torch.cat([p[1] for p in pairs])


@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (128, 8, 1), (64, 6, 2), (128, 32, 1), (64, 40, 2), (128, 2, 2)])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_decode_attention(hd, H, Hk, page):
    """Lengths around the pages' and tiles' ends, none and one, and long ones; stale
    pages and the rows behind a sequence's end hold NaN."""
    from naylis_b200 import attention
    lens = [0, 1, 7, 8, 9, 63, 64, 65, 200, 511, 512, 513, 1500, 2049]
    kp, vp, table, sl, ks, vs = _cache(10, lens, Hk, page, hd, fill=float("nan"))
    q = _rand(9, len(lens), H, hd, scale=2.0)
    want = _decode_exact(q, ks, vs, hd ** -0.5)
    out = attention.decode_attention(q, kp, vp, table, sl)
    _close(out, *want)
    assert torch.equal(out, attention.decode_attention(q, kp, vp, table, sl))
    _close(attention.decode_attention(q, kp, vp, table, sl, max_len=max(lens)), *want)
    # one at a time
    for b in (1, 6, 12):
        _close(attention.decode_attention(q[b:b + 1], kp, vp, table[b:b + 1], sl[b:b + 1], max_len=lens[b]),
               want[0][b:b + 1], want[1][b:b + 1])


@pytest.mark.parametrize("B,hd,H,Hk", [(300, 64, 4, 4), (140, 128, 40, 2), (40, 64, 16, 16), (3, 128, 16, 1)])
def test_decode_attention_spans_of_many_lists(B, hd, H, Hk):
    """More sequences than a CTA has threads and lists that share a CTA, one list over
    many CTAs, more than 16 heads to a key head; lengths of none, one and tiles' ends."""
    from naylis_b200 import attention
    g = torch.Generator().manual_seed(B)
    lens = [[0, 1, 16, 17, -3, 96][i % 6] if i % 2 else int(torch.randint(0, 300, (1,), generator=g)) for i in range(B)]
    lens[B // 2] = 9000
    page = 16
    kp, vp, table, sl, ks, vs = _cache(11, [max(n, 0) for n in lens], Hk, page, hd, fill=float("nan"))
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = _rand(12, B, H, hd, scale=2.0)
    want = _decode_exact(q, ks, vs, hd ** -0.5)
    out = attention.decode_attention(q, kp, vp, table, sl)
    _close(out, *want)
    assert torch.equal(out, attention.decode_attention(q, kp, vp, table, sl))
    # a page outside the cache and a length over max_len spoil their own sequences alone
    table[B // 2, 300] = kp.shape[0]
    table[0, 0] = -1
    sl[0], sl[B - 1] = 5, 9001
    got = attention.decode_attention(q, kp, vp, table, sl, max_len=9000)
    spoilt = torch.zeros(B, dtype=torch.bool, device=DEV)
    spoilt[[0, B // 2, B - 1]] = True
    assert got[spoilt].isnan().all()
    if not spoilt.all():
        _close(got[~spoilt], want[0][~spoilt], want[1][~spoilt])


def test_decode_attention_strides_stream_and_scores():
    """q as a slice of a fused projection, a table with a wider pitch, scores hundreds
    of units apart, on another stream."""
    from naylis_b200 import attention
    lens, H, Hk, hd, page = [700, 33, 1300], 4, 2, 64, 32
    kp, vp, table, sl, ks, vs = _cache(20, lens, Hk, page, hd)
    kp.mul_(12)
    ks = [k * 12 for k in ks]
    wide = torch.full((3, table.shape[1] + 9), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    qkv = _rand(21, 3, H + 2 * Hk, hd, scale=4.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = attention.decode_attention(qkv[:, :H], kp, vp, wide[:, :table.shape[1]], sl, scale=0.7)
    s.synchronize()
    _close(out, *_decode_exact(qkv[:, :H], ks, vs, 0.7))


def test_decode_attention_bad_lengths_and_pages_are_nan():
    from naylis_b200 import attention
    lens, H, Hk, hd, page = [40, 40, 40, 40, 0], 4, 2, 64, 16
    kp, vp, table, sl, ks, vs = _cache(30, lens, Hk, page, hd)
    q = _rand(31, 5, H, hd)
    want = _decode_exact(q, ks, vs, hd ** -0.5)
    table[1, 2] = kp.shape[0]      # outside the cache
    table[2, 0] = -7
    sl[3] = 49                     # longer than the table holds
    sl[4] = -3
    out = attention.decode_attention(q, kp, vp, table, sl)
    assert bool(torch.isnan(out[1:4].float()).all()) and bool((out[4] == 0).all())
    _close(out[:1], want[0][:1], want[1][:1])
    out = attention.decode_attention(q, kp, vp, table, sl, max_len=39)
    assert bool(torch.isnan(out[:4].float()).all()) and bool((out[4] == 0).all())


def test_decode_attention_nan_that_is_seen():
    from naylis_b200 import attention
    lens, H, Hk, hd, page = [600, 600], 4, 2, 64, 16
    kp, vp, table, sl, ks, vs = _cache(40, lens, Hk, page, hd)
    q = _rand(41, 2, H, hd)
    want = _decode_exact(q, ks, vs, hd ** -0.5)
    kp[table[1, 3].long(), 1, 5, 7] = float("nan")
    out = attention.decode_attention(q, kp, vp, table, sl)
    assert bool(torch.isnan(out[1, 2:].float()).all())
    _close(out[1, :2], want[0][1, :2], want[1][1, :2])
    _close(out[0], want[0][0], want[1][0])


def test_cache_beyond_32_bits():
    """Pages whose element offsets pass 2^31 and 2^32."""
    from naylis_b200 import attention
    Hk, page, hd, H = 8, 64, 128, 8
    per = Hk * page * hd
    P = (1 << 32) // per + 40
    kp = torch.empty(P, Hk, page, hd, dtype=torch.bfloat16, device=DEV)
    vp = torch.empty_like(kp)
    n = 150
    ids = [P - 1, (1 << 31) // per, P - 20]
    slots = torch.tensor([ids[t // page] * page + t % page for t in range(n)], device=DEV)
    qkv = _rand(50, n, (H + 2 * Hk) * hd)
    cos = torch.ones(n, hd, device=DEV)
    sin = torch.zeros(n, hd, device=DEV)
    pos = torch.arange(n, device=DEV)
    q, k = attention.rope_append(qkv, cos, sin, pos, kp, vp, slots, n_heads=H, want_k=True)
    x = qkv.view(n, -1, hd)
    assert torch.equal(q, x[:, :H]) and torch.equal(k, x[:, H:H + Hk])
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    out = attention.decode_attention(q[-1:], kp, vp, table, torch.tensor([n], dtype=torch.int32, device=DEV))
    _close(out, *_decode_exact(q[-1:], [k], [x[:, H + Hk:]], hd ** -0.5))


def test_decode_attention_refuses():
    from naylis_b200 import attention
    kp, vp, table, sl, _, _ = _cache(60, [20, 30], 2, 16, 64)
    q = _rand(61, 2, 4, 64)
    assert attention.decode_attention(q[:0], kp, vp, table[:0], sl[:0]).shape == (0, 4, 64)
    bad = [(q.float(), kp, vp, table, sl), (q, kp.float(), vp.float(), table, sl), (q, kp, vp[:1], table, sl),
           (q, kp, vp, table.long(), sl), (q, kp, vp, table, sl.long()), (q, kp, vp, table[:1], sl),
           (q, kp, vp, table, sl[:1]), (q[:, :3], kp, vp, table, sl), (q[..., :32], kp, vp, table, sl),
           (q, kp[:, :, :12], vp[:, :, :12], table, sl), (q, kp.transpose(1, 2), vp.transpose(1, 2), table, sl),
           (q, kp, vp, table.cpu(), sl), (q.clone().requires_grad_(True), kp, vp, table, sl)]
    for args in bad:
        with pytest.raises(RuntimeError):
            attention.decode_attention(*args)
    for kw in ({"max_len": -1}, {"max_len": 10 ** 6}, {"scale": float("inf")}, {"scale": 0.0}, {"scale": -1.0}):
        with pytest.raises(RuntimeError):
            attention.decode_attention(q, kp, vp, table, sl, **kw)


# ------------------------------------------------------------------ rope_append
@pytest.mark.parametrize("hd,H,Hk,page,T", [(64, 4, 4, 16, 1), (64, 6, 2, 8, 37), (128, 8, 1, 64, 300),
                                            (128, 2, 2, 256, 5), (64, 16, 16, 32, 64)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_rope_append(hd, H, Hk, page, T, itype):
    from naylis_b200 import attention
    from naylis_b200.decoder import apply_rope, rope_tables
    cos, sin = rope_tables(1000, hd, 500000.0, DEV)
    wide = _rand(70, T, (H + 2 * Hk) * hd + 8)
    qkv = wide[:, :(H + 2 * Hk) * hd]
    g = torch.Generator().manual_seed(71)
    pos = torch.randint(0, 1000, (T,), generator=g).to(itype).to(DEV)
    P = T // page + 3
    slots = torch.randperm(P * page, generator=g)[:T].to(itype).to(DEV)
    slots[T // 2] = -1 if T > 1 else slots[0]
    kp, vp = _rand(72, P, Hk, page, hd), _rand(73, P, Hk, page, hd)
    want_kp, want_vp = kp.clone(), vp.clone()
    x = qkv.reshape(T, H + 2 * Hk, hd)
    rot = apply_rope(x[:, :H + Hk].transpose(0, 1), cos[pos.long()], sin[pos.long()]).transpose(0, 1).bfloat16()
    live = slots >= 0
    s = slots[live].long()
    want_kp[s // page, :, s % page] = rot[live, H:]
    want_vp[s // page, :, s % page] = x[live, H + Hk:]
    q, k = attention.rope_append(qkv, cos, sin, pos, kp, vp, slots, n_heads=H, want_k=True)
    assert torch.equal(q, rot[:, :H]) and torch.equal(k, rot[:, H:])
    assert torch.equal(kp, want_kp) and torch.equal(vp, want_vp)
    q2, none = attention.rope_append(qkv, cos, sin, pos, kp, vp, slots, n_heads=H)
    assert none is None and torch.equal(q2, q)


def test_rope_append_out_of_range_and_refusals():
    from naylis_b200 import attention
    from naylis_b200.decoder import rope_tables
    hd, H, Hk, page, T = 64, 4, 2, 16, 6
    cos, sin = rope_tables(10, hd, 500000.0, DEV)
    qkv = _rand(80, T, (H + 2 * Hk) * hd)
    kp, vp = torch.zeros(2, Hk, page, hd, dtype=torch.bfloat16, device=DEV), None
    vp = torch.zeros_like(kp)
    pos = torch.tensor([0, 10, -1, 9, 3, 4], device=DEV)
    slots = torch.tensor([0, 1, 2, 32, -5, 1 << 40], device=DEV)
    q, k = attention.rope_append(qkv, cos, sin, pos, kp, vp, slots, n_heads=H, want_k=True)
    nan = torch.isnan(q.float()).flatten(1).all(1)
    assert nan.tolist() == [False, True, True, False, False, False]
    assert torch.equal(vp[0, :, :3].transpose(0, 1), qkv.view(T, -1, hd)[:3, H + Hk:])
    assert int((vp != 0).flatten(2).any(-1).sum()) == 3 * Hk or bool((vp[0, :, 3:] == 0).all())
    assert bool((vp[1] == 0).all()) and bool((kp[1] == 0).all()) and bool((kp[0, :, 3:] == 0).all())
    e = attention.rope_append(qkv[:0], cos, sin, pos[:0], kp, vp, slots[:0], n_heads=H, want_k=True)
    assert e[0].shape == (0, H, hd) and e[1].shape == (0, Hk, hd)
    for args, kw in [((qkv.float(), cos, sin, pos, kp, vp, slots), {}), ((qkv, cos.double(), sin, pos, kp, vp, slots), {}),
                     ((qkv, cos, sin[:5], pos, kp, vp, slots), {}), ((qkv, cos, sin, pos[:5], kp, vp, slots), {}),
                     ((qkv, cos, sin, pos, kp, vp, slots.float()), {}), ((qkv[:, 1:], cos, sin, pos, kp, vp, slots), {}),
                     ((qkv, cos, sin, pos, kp, vp, slots), {"n_heads": 3}), ((qkv, cos, sin, pos, kp, vp[:1], slots), {}),
                     ((qkv, cos, sin, pos, kp[..., :32], vp[..., :32], slots), {})]:
        with pytest.raises(RuntimeError):
            attention.rope_append(*args, **{"n_heads": H, **kw})
