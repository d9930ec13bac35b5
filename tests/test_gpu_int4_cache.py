"""GPU tests of the 4-bit cache (rope_append_int4, decode_attention_int4) against their
definitions.

rope_append_int4 is exact: the rotation is rope_append's bit for bit, and scale, zero
and numbers follow from fp32 operations that torch rounds the same way.

Tolerance of decode_attention_int4, per element, with A = sum_t p_t (|zero| + n scale),
which bounds |out| and every partial sum: the output is rounded to bf16 (2^-8 of |out|),
the weights p_t scale to fp16 (2^-11 of what they weigh, at most of A; below 2^-24 of the
greatest weight they lose bits, 2^-38 a key), exponentials and scores are within 2^-12 (of
A) for scores up to about 100, fp32 sums far below. So |got - exact| <= 2^-8 |exact| + 2^-10 A;
2^-40 covers A = 0.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
NAN = float("nan")


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(DEV)


def _cache(seed, pages, Hk, page, hd):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randint(0, 256, (pages, Hk, page, hd // 2), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    s = torch.randn(pages, Hk, page, hd // 64, 4, generator=g) * 0.1
    s[..., 0::2] = 0.1 + s[..., 0::2].abs()
    s[..., 1::2] -= 7.5 * s[..., 0::2]
    return k, v, s.to(torch.bfloat16).to(DEV)


def _values(raw, scales, i):
    """What rows (..., hd / 2) of pages stand for, with their (..., groups, 4) scales, in 64 bits."""
    n = torch.stack((raw & 15, raw >> 4), -1).flatten(-2).double().unflatten(-1, (-1, 64))
    s = scales.double()
    return (n * s[..., 2 * i, None] + s[..., 2 * i + 1, None]).flatten(-2), \
        (n * s[..., 2 * i, None] + s[..., 2 * i + 1, None].abs()).flatten(-2)


def _exact(q, cache, table, lens, news, scale):
    k_pages, v_pages, scales = cache
    B, n, H, hd = q.shape
    Hk, page = k_pages.shape[1:3]
    G = H // Hk
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    A = torch.zeros_like(out)
    for b in range(B):
        if lens[b] <= 0:
            continue
        t = torch.arange(lens[b], device=DEV)
        at, off = table[b].long()[t // page], t % page
        k, _ = _values(k_pages[at, :, off], scales[at, :, off], 0)
        v, va = _values(v_pages[at, :, off], scales[at, :, off], 1)
        for j in range(news[b]):
            e = lens[b] - news[b] + j + 1
            if e <= 0:
                continue
            qq = q[b, j].double().view(Hk, G, hd)
            p = torch.softmax(torch.einsum("hgd,thd->hgt", qq, k[:e]) * scale, -1)
            out[b, j] = torch.einsum("hgt,thd->hgd", p, v[:e]).reshape(H, hd)
            A[b, j] = torch.einsum("hgt,thd->hgd", p, va[:e]).reshape(H, hd)
    return out, A


def _close(got, out, A):
    assert bool(torch.isfinite(got).all())
    err = (got.double() - out).abs()
    worst = float((err - 2.0 ** -8 * out.abs() - 2.0 ** -10 * A).max())
    assert worst <= 2.0 ** -40, (worst, float(err.max()))


def _table(seed, lens, page, spare=3):
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    o = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[o:o + n]
        o += n
    return total, table.to(DEV)


def _spoil_ends(cache, table, lens, page):
    """NaN scales and full bytes in the rows behind each sequence's end, in its last page."""
    k, v, s = cache
    for b, n in enumerate(lens):
        if n > 0 and n % page:
            p = int(table[b, n // page])
            s[p, :, n % page:] = NAN
            k[p, :, n % page:] = 255
            v[p, :, n % page:] = 255


def _case(hd, H, Hk, page, lens, n, news=None, seed=0, qscale=2.0):
    total, table = _table(seed, lens, page)
    cache = _cache(seed + 1, total, Hk, page, hd)
    _spoil_ends(cache, table, lens, page)
    q = _rand(seed + 2, len(lens), n, H, hd, scale=qscale)
    return q, cache, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def _run(q, cache, table, lens, **kw):
    from naylis_b200 import attention
    return attention.decode_attention_int4(q, *cache, table, lens, **kw)


LENS = [[1], [31, 32, 33], [577], [128, 0, 5, 1000, 64], [4097, 1, 300], [20000, 3, 70]]


# ------------------------------------------------------------------ decode
@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (64, 16, 16), (128, 8, 2), (128, 16, 1), (64, 20, 1), (128, 5, 1)])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_one_new_token(hd, H, Hk, page, lens):
    q, cache, table, sl = _case(hd, H, Hk, page, lens, 1, seed=hd + H + page)
    got = _run(q, cache, table, sl)
    _close(got, *_exact(q, cache, table, lens, [1] * len(lens), hd ** -0.5))
    assert torch.equal(got, _run(q, cache, table, sl))


@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (64, 6, 2), (128, 8, 2), (128, 8, 1), (64, 40, 2)])
@pytest.mark.parametrize("n", [2, 3, 5, 8, 17, 64])
@pytest.mark.parametrize("lens", [[64, 65, 100], [700, 0, 5, 64], [9000, 200]], ids=str)
def test_several_new_tokens(hd, H, Hk, n, lens):
    """Causal among themselves; a sequence shorter than its new tokens has rows without keys."""
    q, cache, table, sl = _case(hd, H, Hk, 16, lens, n, seed=hd + H + n)
    got = _run(q, cache, table, sl, scale=0.11)
    _close(got, *_exact(q, cache, table, lens, [n] * len(lens), 0.11))
    news = [(3 * i + n // 2) % (n + 1) for i in range(len(lens))]
    new_lens = torch.tensor(news, dtype=torch.int32, device=DEV)
    got = _run(q, cache, table, sl, new_lens=new_lens)
    _close(got, *_exact(q, cache, table, lens, news, hd ** -0.5))
    for b, m in enumerate(news):
        assert not got[b, m:].any()


@pytest.mark.parametrize("hd,H,Hk,n", [(64, 16, 16, 1), (128, 16, 4, 1), (128, 16, 4, 5)])
def test_a_busy_batch(hd, H, Hk, n):
    """Spans that begin and end inside lists, and more lists than CTAs."""
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.exp(torch.rand(70, generator=g) * 8.2)]
    q, cache, table, sl = _case(hd, H, Hk, 32, lens, n, seed=9)
    got = _run(q, cache, table, sl)
    _close(got, *_exact(q, cache, table, lens, [n] * len(lens), hd ** -0.5))
    assert torch.equal(got, _run(q, cache, table, sl))


@pytest.mark.parametrize("hd", [64, 128])
def test_a_long_sequence(hd):
    lens = [131072, 100001]
    q, cache, table, sl = _case(hd, 8, 2, 64, lens, 2, seed=3)
    _close(_run(q, cache, table, sl), *_exact(q, cache, table, lens, [2, 2], hd ** -0.5))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,n", [(2, 1), (8, 1), (2, 7)])
def test_a_long_mean(hd, H, n):
    """All keys alike (a query of 0): the mean of 131072 values, near 0 with numbers around the
    middle of their groups. Weights are the values' scales, exact in fp16; a warp's sums, of up
    to all keys of a list, may be off by 2^-20 of what they sum (fp32, rounded towards zero
    within a few tiles): 15 scales, so 2^-16 of the greatest scale, twice for the two sums."""
    lens = [131072]
    q, (k, v, s), table, sl = _case(hd, H, 2, 64, lens, n, seed=12)
    g = torch.Generator().manual_seed(5)
    num = torch.randn(2, *v.shape, generator=g).mul(3.2).add(7.5).round().clamp(0, 15).to(torch.uint8).to(DEV)
    cache = (k, num[0] | num[1] << 4, s)
    s[..., 3] = (-7.5 * s[..., 2].float()).to(torch.bfloat16)
    got = _run(q * 0, cache, table, sl)
    out, A = _exact(q * 0, cache, table, lens, [n], 1.0)
    worst = float(((got.double() - out).abs() - 2.0 ** -8 * out.abs()).max())
    assert worst <= 2.0 ** -15 * float(s[..., 2].max()), worst


@pytest.mark.parametrize("lens", [[300, 40], [30000, 257]], ids=str)
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_of_very_different_size(hd, lens):
    """Value scales that rise along the sequence by powers of ten, fall, and are 0 or tiny."""
    q, cache, table, sl = _case(hd, 4, 2, 16, lens, 3, seed=11)
    k, v, s = cache
    t = torch.arange(s.shape[0] * 16, device=DEV).view(-1, 1, 16)
    for f in (torch.pow(10.0, (t % 977).float() / 100 - 5), torch.pow(10.0, 5 - (t % 977).float() / 100),
              torch.where(t % 3 == 0, 0.0, 1.0), torch.full_like(t, 1, dtype=torch.float32) * 1e-30,
              torch.full_like(t, 1, dtype=torch.float32) * 1e30):
        s2 = s.clone()
        s2[..., 2:] = (s[..., 2:].float() * f[..., None, None]).to(torch.bfloat16)
        got = _run(q, (k, v, s2), table, sl)
        out, A = _exact(q, (k, v, s2), table, lens, [3] * len(lens), hd ** -0.5)
        _close(got, out, A)


@pytest.mark.parametrize("hd", [64, 128])
def test_wide_scores(hd):
    """Scores hundreds of units apart, rising along the sequence (the maximum moves at every
    tile), and falling; queries from tiny to huge."""
    lens = [3000]
    q, cache, table, sl = _case(hd, 2, 2, 16, lens, 2, seed=4)
    k, v, s = cache
    order = torch.empty(s.shape[0], dtype=torch.long, device=DEV)
    order[table[0].long()] = torch.arange(table.shape[1], device=DEV)
    pos = (order[:, None] * 16 + torch.arange(16, device=DEV)).float()
    k &= 0
    for ramp in (pos / 10 - 150, 150 - pos / 10):
        s2 = s.clone()
        s2[..., 0] = 0
        s2[..., 1] = ramp[:, None, :, None].to(torch.bfloat16)
        ones = torch.ones_like(q)
        got = _run(ones, (k, v, s2), table, sl, scale=1.0 / hd)
        _close(got, *_exact(ones, (k, v, s2), table, lens, [2], 1.0 / hd))
    cache = _cache(77, s.shape[0], 2, 16, hd)
    for f in (1e-30, 1e-6, 1e6, 1e20):
        qf = (q.float() * f).to(torch.bfloat16)
        got = _run(qf, cache, table, sl, scale=min(1.0, 0.3 / f))
        _close(got, *_exact(qf, cache, table, lens, [2], min(1.0, 0.3 / f)))
    zero = torch.zeros_like(q)
    _close(_run(zero, cache, table, sl), *_exact(zero, cache, table, lens, [2], 1.0))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,n", [(2, 1), (8, 1), (2, 5), (8, 5)])
@pytest.mark.parametrize("size", [1e3, 1e9, 1e25])
@pytest.mark.parametrize("lens", [[9000, 300], [400, 130]], ids=str)
def test_huge_scores(hd, H, n, size, lens):
    """Scores far beyond where fp32 has fractions, the greatest 1 % and more above all others: it has all the weight.
    Products and sums are within 2^-18 of a score, so no other comes near it."""
    q, (k, v, s), table, sl = _case(hd, H, 2, 16, lens, n, seed=14)
    s = torch.nan_to_num(s.float(), nan=0.5)
    g = torch.Generator().manual_seed(15)
    s[..., 0] = 0
    s[..., 1] = (torch.rand(s.shape[:3], generator=g).to(DEV) * 150 + 30)[..., None]
    for b, at in ((0, 7 * lens[0] // 9), (1, 117)):
        s[int(table[b, at // 16]), :, at % 16, :, 1] = 187.0
    s = s.to(torch.bfloat16)
    q = torch.full_like(q, size) * (1 + torch.arange(H, device=DEV)[:, None] / 16).to(torch.bfloat16)
    got = _run(q, (k, v, s), table, sl, scale=0.37)
    _close(got, *_exact(q, (k, v, s), table, lens, [n, n], 0.37))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[200, 40], [20000, 257]], ids=str)
def test_hidden_groups_stay_hidden(hd, lens):
    """The last draft's key or value stands for NaN: the tokens before it do not see it."""
    n = 4
    q, cache, table, sl = _case(hd, 8, 2, 16, lens, n, seed=6)
    k, v, s = cache
    want, A = _exact(q, cache, table, lens, [n] * 2, hd ** -0.5)
    at = [(int(table[b, (m - 1) // 16]), (m - 1) % 16) for b, m in enumerate(lens)]
    for i in range(4):
        s2 = s.clone()
        for p, o in at:
            s2[p, 1, o, 0, i] = NAN
        got = _run(q, (k, v, s2), table, sl)
        hit = torch.zeros_like(got, dtype=torch.bool)
        if i < 2:
            hit[:, n - 1, 4:] = True
        else:
            hit[:, n - 1, 4:, :64] = True
        _close(got[~hit], want[~hit], A[~hit])
        assert bool(torch.isnan(got[hit]).all())


@pytest.mark.parametrize("big", [False, True])
def test_what_is_not_there_is_nan(big):
    lens = [20000 if big else 300, 100, 90, 80, 70]
    q, cache, table, sl = _case(64, 4, 4, 16, lens, 3, seed=8)
    want, A = _exact(q, cache, table, lens, [3] * 5, 0.125)
    ok = [0, 2, 4]
    for bad in (-1, 1 << 30, cache[0].shape[0]):
        t2 = table.clone()
        t2[1, 2] = bad
        got = _run(q, cache, t2, sl)
        assert bool(torch.isnan(got[1]).all())
        _close(got[ok], want[ok], A[ok])
    got = _run(q, cache, table, sl, max_len=max(lens) - 1)      # sequence 0 is longer than the caller says
    assert bool(torch.isnan(got[0]).all())
    _close(got[2:], want[2:], A[2:])
    news = torch.tensor([3, 4, 3, -1, 3], dtype=torch.int32, device=DEV)
    got = _run(q, cache, table, sl, new_lens=news)
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[3]).all())
    _close(got[ok], want[ok], A[ok])
    q2 = q.clone()
    q2[2, 1, 1, 3] = float("inf")
    q2[4, 0, 0, 0] = NAN
    got = _run(q2, cache, table, sl)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[2, 1, 1] = hit[4, 0, 0] = True
    assert bool(torch.isnan(got[hit]).all())
    _close(got[~hit], want[~hit], A[~hit])
    none = torch.tensor([0, -5, -2147483648, 0, 0], dtype=torch.int32, device=DEV)
    assert not _run(q, cache, table, none).any()


@pytest.mark.parametrize("big", [False, True])
def test_other_streams_strides_and_graphs(big):
    from naylis_b200 import attention
    lens = [20000 if big else 300, 100]
    _, cache, table, sl = _case(64, 4, 2, 16, lens, 2, seed=8)
    wide = _rand(1, 2, 2, 6, 64, scale=2.0)
    q = wide[:, :, :4]                                       # a slice of a wider projection
    want, A = _exact(q, cache, table, lens, [2, 2], 0.125)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, cache, table, sl)
    side.synchronize()
    _close(got, want, A)
    flipped = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(_run(flipped, cache, table, sl), got)
    wide_table = torch.cat((table, table), 1)[:, :table.shape[1]]
    assert torch.equal(_run(q, cache, wide_table, sl), got)
    # two captured graphs, replayed in turn and at once: a workspace each
    other = _rand(2, 2, 2, 4, 64)
    graphs = []
    for x in (q, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attention.decode_attention_int4(x, *cache, table, sl)
        graphs.append((g, out))
    for _ in range(3):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], got) and torch.equal(graphs[1][1], _run(other, cache, table, sl))


# ------------------------------------------------------------------ append
def _plain_int4(x):
    y = x.float().unflatten(-1, (-1, 64))
    zero, most = y.amin(-1), y.amax(-1)
    span = most - zero
    step = (span * (1.0 / 15.0)).to(torch.bfloat16).float()
    odd = ~torch.isfinite(y).all(-1) | ~torch.isfinite(span)
    step, zero = torch.where(odd, NAN, step), torch.where(odd, NAN, zero)
    n = torch.where(step[..., None] > 0, (y - zero[..., None]) / step[..., None], 0.0).round().clamp(0, 15)
    stands = (n * step[..., None] + zero[..., None]).flatten(-2).to(torch.bfloat16)
    return n.flatten(-2).to(torch.uint8), step.to(torch.bfloat16), zero.to(torch.bfloat16), stands


def _same(a, b):
    """Equal values; NaN is NaN (whatever its bits) and -0 is 0."""
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def _check_append(qkv, cos, sin, pos, slots, H, Hk, hd, page, pages, seed=0):
    from naylis_b200 import attention
    T = qkv.shape[0]
    cache = _cache(seed, pages, Hk, page, hd)
    before = [t.clone() for t in cache]
    q, k, v = attention.rope_append_int4(qkv, cos, sin, pos, *cache, slots, n_heads=H, want_kv=True)
    kp = torch.zeros(pages, Hk, page, hd, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    q0, k0 = attention.rope_append(qkv, cos, sin, pos, kp, vp, slots, n_heads=H, want_k=True)
    assert _same(q, q0) and q.shape == (T, H, hd)
    v0 = qkv.reshape(T, H + 2 * Hk, hd)[:, H + Hk:]
    want = [t.clone() for t in before]
    here = ((slots >= 0) & (slots < pages * page)).nonzero()[:, 0]
    at, off = slots[here].long() // page, slots[here].long() % page
    for i, (x, got) in enumerate(((k0, k), (v0, v))):
        n, step, zero, stands = _plain_int4(x)
        assert _same(got, stands)
        want[i][at, :, off] = (n[..., 0::2] | n[..., 1::2] << 4)[here]
        want[2][at, :, off, :, 2 * i] = step[here]
        want[2][at, :, off, :, 2 * i + 1] = zero[here]
    assert torch.equal(cache[0], want[0]) and torch.equal(cache[1], want[1]) and _same(cache[2], want[2])
    again = [t.clone() for t in before]
    q2, k2, v2 = attention.rope_append_int4(qkv, cos, sin, pos, *again, slots, n_heads=H)
    assert k2 is None and v2 is None and _same(q2, q)
    assert torch.equal(again[0], cache[0]) and torch.equal(again[1], cache[1]) and _same(again[2], cache[2])


def _tables(n, hd):
    from naylis_b200.decoder import rope_tables
    return rope_tables(n, hd, 500000.0, DEV)


@pytest.mark.parametrize("hd,H,Hk", [(64, 16, 16), (128, 16, 4), (64, 3, 1), (128, 5, 5), (64, 10, 2)])
@pytest.mark.parametrize("T,page", [(0, 16), (1, 8), (5, 16), (333, 64), (5000, 32)])
def test_append(hd, H, Hk, T, page):
    pages = -(-T // page) + 2
    g = torch.Generator().manual_seed(T + hd)
    qkv = _rand(T + H, T, (H + 2 * Hk) * hd)
    slots = torch.randperm(pages * page, generator=g)[:T].to(DEV)
    pos = torch.randint(0, 6000, (T,), generator=g).to(DEV)
    if T > 3:
        slots[1], slots[3] = -1, pages * page            # padding
    cos, sin = _tables(6000, hd)
    _check_append(qkv, cos, sin, pos, slots, H, Hk, hd, page, pages)
    _check_append(qkv, cos, sin, pos.int(), slots.int(), H, Hk, hd, page, pages, seed=1)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_odd_values(hd):
    """Groups of one value, of zeros, of tiny and huge values, a range beyond fp32, NaN and
    infinities; positions outside the tables; a strided projection."""
    H, Hk, T, page = 2, 2, 40, 16
    wide = _rand(3, T, 2 * (H + 2 * Hk) * hd)
    qkv = wide[:, :(H + 2 * Hk) * hd]
    x = qkv.view(T, -1, hd)
    x[1] = 0.0
    x[2] = -3.5
    x[3] *= 1e-39
    x[4] *= 1e37
    x[5, :, 0], x[5, :, 1] = 3.3e38, -3.3e38
    x[6, :, 7] = NAN
    x[7, :, hd - 1] = float("inf")
    x[8, :, 33] = float("-inf")
    x[9, :, 5] = 1e20
    x[10] = x[10].abs() + 100.0
    x[11, :, 1::2] = -0.0
    x[11, :, 0::2] = 0.0
    x[12] = torch.arange(hd, device=DEV).to(torch.bfloat16) % 16
    x[13] = (torch.arange(hd, device=DEV) % 16).to(torch.bfloat16) * 0.5 + 0.25
    pos = torch.arange(T, device=DEV)
    pos[20], pos[21] = -1, 64
    slots = torch.arange(T, device=DEV).flip(0)
    cos, sin = _tables(64, hd)
    _check_append(qkv, cos, sin, pos, slots, H, Hk, hd, page, 3)
    cos, sin = torch.ones_like(cos), torch.zeros_like(sin)          # the keys' own values
    _check_append(qkv, cos, sin, pos, slots, H, Hk, hd, page, 3)


def test_append_then_attend():
    """Prefill, then steps of drafts: the cache's numbers come back as attention sees them."""
    from naylis_b200 import attention
    H, Hk, hd, page = 8, 2, 64, 16
    cos, sin = _tables(400, hd)
    cache = _cache(0, 30, Hk, page, hd)
    table = torch.arange(30, device=DEV, dtype=torch.int32).flip(0)[None].contiguous()
    ks, vs, done = [], [], 0
    for n in (200, 1, 5, 3):
        qkv = _rand(n, n, (H + 2 * Hk) * hd)
        pos = torch.arange(done, done + n, device=DEV)
        slots = table[0].long()[pos // page] * page + pos % page
        q, k, v = attention.rope_append_int4(qkv, cos, sin, pos, *cache, slots, n_heads=H, want_kv=True)
        ks.append(k)
        vs.append(v)
        done += n
        if n <= 64:
            sl = torch.tensor([done], dtype=torch.int32, device=DEV)
            got = attention.decode_attention_int4(q[None], *cache, table, sl)[0]
            _close(got[None], *_exact(q[None], cache, table, [done], [n], hd ** -0.5))
            # prompt_attention over the values that were handed back (rounded to bf16: 2^-8 of each
            # more, in scores of up to 8 units 2^-5, and its own weights' rounding)
            plan = attention.PromptPlan([n], [done], device=DEV)
            o = attention.prompt_attention(q, torch.cat(ks), torch.cat(vs), plan)
            assert float((o.float() - got.float()).abs().max()) < 2.0 ** -4 * float(got.float().abs().max())


def test_refusals():
    from naylis_b200 import attention
    q, cache, table, sl = _case(64, 4, 2, 16, [100, 3], 2, seed=1)
    k, v, s = cache
    dec = attention.decode_attention_int4
    app = attention.rope_append_int4
    for bad in (lambda: dec(q.float(), k, v, s, table, sl), lambda: dec(q[:, 0], k, v, s, table, sl),
                lambda: dec(q, k.float(), v, s, table, sl), lambda: dec(q, k, v[:1], s, table, sl),
                lambda: dec(q, k, v, s.float(), table, sl), lambda: dec(q, k, v, s[..., :2], table, sl),
                lambda: dec(q, k[:, :, :12], v[:, :, :12], s[:, :, :12], table, sl),
                lambda: dec(q[..., :32], k, v, s, table, sl), lambda: dec(q[:, :, :3], k, v, s, table, sl),
                lambda: dec(q[:, :0], k, v, s, table, sl), lambda: dec(q.repeat(1, 33, 1, 1), k, v, s, table, sl),
                lambda: dec(q, k, v, s, table.long(), sl), lambda: dec(q, k, v, s, table, sl.long()),
                lambda: dec(q, k, v, s, table, sl, new_lens=sl[:1]), lambda: dec(q, k, v, s, table, sl, max_len=10 ** 6),
                lambda: dec(q, k, v, s, table, sl, new_lens=sl.long()), lambda: dec(q, k, v, s, table, sl, scale=0.0),
                lambda: dec(q, k, v, s, table, sl.cpu()), lambda: dec(q, k.cpu(), v.cpu(), s, table, sl),
                lambda: dec(q.requires_grad_(True), k, v, s, table, sl)):
        with pytest.raises(RuntimeError):
            bad()
    cos, sin = _tables(8, 64)
    x = _rand(0, 2, 8 * 64)
    i = torch.arange(2, device=DEV)
    app(x, cos, sin, i, k, v, s, i, n_heads=4)
    for bad in (lambda: app(x, cos, sin, i, k, v, s, i, n_heads=3), lambda: app(x.float(), cos, sin, i, k, v, s, i, n_heads=4),
                lambda: app(x, cos.double(), sin, i, k, v, s, i, n_heads=4), lambda: app(x, cos, sin, i[:1], k, v, s, i, n_heads=4),
                lambda: app(x, cos, sin, i, k, v, s, i.float(), n_heads=4), lambda: app(x, cos, sin, i, k, v, s[:1], i, n_heads=4),
                lambda: app(x, cos, sin, i, k.to(torch.int8), v, s, i, n_heads=4)):
        with pytest.raises(RuntimeError):
            bad()
    assert dec(q[:0].detach(), k, v, s, table[:0], sl[:0]).shape == (0, 2, 4, 64)
