"""GPU tests of decode_attention_int4 at the ends of its range: scales, queries and lengths far
from the usual ones. Tolerances, where not said otherwise, are test_gpu_int4_cache's: the
weights' fp16 numbers lose bits below 2^-21 of the row's greatest product of weight and
scale, 2^-32 of it and 15 numbers a key, which 2^-10 A contains up to 2^18 keys. (No floor
under the tolerance: outputs may be as small as their values.)"""
import pytest
import torch

from test_gpu_int4_cache import DEV, _case, _exact, _run

pytestmark = pytest.mark.gpu


def _close(got, out, A):
    assert bool(torch.isfinite(got).all())
    over = (got.double() - out).abs() / (2.0 ** -8 * out.abs() + 2.0 ** -10 * A + 2.0 ** -126)
    assert float(over.max()) <= 1.0, (float(over.max()), over.argmax())

# ------------------------------------------------------------------ scales that do not count
FORMS = [(2, 2, 4), (8, 2, 4), (4, 2, 2), (2, 1, 8), (16, 2, 4)]      # lists of 4, 8 and more rows


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,n", FORMS)
@pytest.mark.parametrize("lens", [[200, 40], [20000, 257]], ids=str)
def test_hidden_scales_stay_hidden(hd, H, Hk, n, lens):
    """The last draft's key or value has a huge scale or zero: the tokens before it do not see it."""
    q, cache, table, sl = _case(hd, H, Hk, 16, lens, n, seed=21)
    k, v, s = cache
    want, A = _exact(q, cache, table, lens, [n] * 2, hd ** -0.5)
    at = [(int(table[b, (m - 1) // 16]), (m - 1) % 16) for b, m in enumerate(lens)]
    for big in (1e8, 1e20, 1e30, float("inf")):
        for i in range(4):
            s2 = s.clone()
            for p, o in at:
                s2[p, :, o, :, i] = big
            got = _run(q, (k, v, s2), table, sl)
            _close(got[:, :n - 1], want[:, :n - 1], A[:, :n - 1])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,n", [(2, 2, 1), (4, 1, 1)] + FORMS)
@pytest.mark.parametrize("lens", [[300, 130], [20000, 257]], ids=str)
@pytest.mark.parametrize("jump", [False, True])
def test_scales_without_weight(hd, H, Hk, n, lens, jump):
    """Keys whose values have a huge scale and whose score is 200 below the others': their weight of
    e^-200 is nothing, and the others keep theirs. Jump: they weigh much until, two thirds
    along the sequence, the scores rise by 200."""
    q, (k, v, s), table, sl = _case(hd, H, Hk, 16, lens, n, seed=22)
    q = torch.ones_like(q)
    k = torch.zeros_like(k)
    s = torch.nan_to_num(s.float(), nan=0.5)
    g = torch.Generator().manual_seed(23)
    s[..., 0] = 0
    s[..., 1] = torch.rand(s.shape[:3], generator=g).to(DEV)[..., None] * 4 - 2      # a key's score, with scale 1 / hd
    for big in (1e8, 1e11, 1e30):
        s2 = s.clone()
        for b, m in enumerate(lens):
            t = torch.arange(m, device=DEV)
            pages = table[b].long()[t // 16]
            if jump:
                low = t < 2 * m // 3
                s2[pages[low], :, (t % 16)[low], :, 1] -= 200.0
            for o in (0, 5, 61, m // 3, m // 2, 2 * m // 3 - 1):
                p = int(table[b, o // 16])
                s2[p, :, o % 16, :, 2:] = big
                if not jump:
                    s2[p, :, o % 16, :, 1] = -200.0
        s2 = s2.to(torch.bfloat16)
        got = _run(q, (k, v, s2), table, sl, scale=1.0 / hd)
        _close(got, *_exact(q, (k, v, s2), table, lens, [n] * len(lens), 1.0 / hd))
        assert torch.equal(got, _run(q, (k, v, s2), table, sl, scale=1.0 / hd))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,n", [(2, 2, 1), (2, 2, 4), (8, 2, 4)])
def test_products_that_rise_and_fall(hd, H, Hk, n):
    """Scales that fall by powers of ten while the scores rise, and the other way: the weights' products
    with them stay, rise or fall."""
    lens = [3000]
    q, (k, v, s), table, sl = _case(hd, H, Hk, 16, lens, n, seed=24)
    q = torch.ones_like(q)
    k = torch.zeros_like(k)
    order = torch.empty(s.shape[0], dtype=torch.long, device=DEV)
    order[table[0].long()] = torch.arange(table.shape[1], device=DEV)
    pos = ((order[:, None] * 16 + torch.arange(16, device=DEV)).float() / 3000)[:, None, :, None]
    s = torch.nan_to_num(s.float(), nan=0.5)
    for score, size in ((60.0, -60.0), (-60.0, 60.0), (60.0, 20.0), (-60.0, -20.0), (20.0, -60.0), (0.0, 80.0), (0.0, -80.0)):
        s2 = s.clone()
        s2[..., 0] = 0
        s2[..., 1] = score * pos
        s2[..., 2:] *= torch.exp(size * pos[..., None])
        s2 = s2.to(torch.bfloat16)
        got = _run(q, (k, v, s2), table, sl, scale=1.0 / hd)
        _close(got, *_exact(q, (k, v, s2), table, lens, [n], 1.0 / hd))


@pytest.mark.parametrize("H,Hk,n", [(2, 2, 1), (2, 2, 4), (8, 2, 4)])
def test_scales_that_are_not_finite(H, Hk, n):
    """An infinite scale of a value that is seen makes its group's outputs inf or NaN, and no others."""
    lens = [700]
    q, (k, v, s), table, sl = _case(128, H, Hk, 16, lens, n, seed=25)
    want, A = _exact(q, (k, v, s), table, lens, [n], 128 ** -0.5)
    for o in (3, 690):
        s2 = s.clone()
        s2[int(table[0, o // 16]), 0, o % 16, 1, 2] = float("inf")
        got = _run(q, (k, v, s2), table, sl)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:, :, :H // Hk, 64:] = True
        _close(got[~hit], want[~hit], A[~hit])
        assert not bool(torch.isfinite(got[hit]).any())

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,n", [(2, 2, 1), (2, 2, 4), (8, 2, 4)])
@pytest.mark.parametrize("size", [2.0 ** 124, 1e36, 1e-36, 2.0 ** -126])
def test_scales_at_the_ends(hd, H, Hk, n, size):
    """The greatest scale that a finite range has, and the least normal one; few keys, whose sums stay in fp32."""
    lens = [2, 1, 0]
    q, (k, v, s), table, sl = _case(hd, H, Hk, 16, lens, n, seed=26, qscale=0.1)
    s2 = torch.nan_to_num(s.float(), nan=0.5)
    s2[..., 2], s2[..., 3] = size, -3.75 * size
    s2 = s2.to(torch.bfloat16)
    v = v & 0x77      # numbers up to 7: values within 3.75 scales of 0
    got = _run(q, (k, v, s2), table, sl)
    _close(got, *_exact(q, (k, v, s2), table, lens, [n] * 3, hd ** -0.5))


# ------------------------------------------------------------------ queries of any size
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,n", [(2, 2, 1), (2, 2, 4), (8, 2, 4)])
@pytest.mark.parametrize("f", [3e37, 1e36, 1e34, 1e31, 1e-24, 1e-28, 1e-32, 1e-36, 1e-38, 2e-39])
def test_queries_of_any_size(hd, H, Hk, n, f):
    """Queries up to the greatest bf16 number and down to its subnormals, with scales that bring their
    scores back to a few units."""
    lens = [1000, 70]
    q, cache, table, sl = _case(hd, H, Hk, 16, lens, n, seed=31)
    q = (q.float() * f).clamp(-3e38, 3e38).to(torch.bfloat16)
    scale = min(0.3 / f, 2e38)
    got = _run(q, cache, table, sl, scale=scale)
    want, A = _exact(q, cache, table, lens, [n] * 2, scale)
    _close(got, want, A)
    # the scores count: the mean of the values is something else
    mean, _ = _exact(q * 0, cache, table, lens, [n] * 2, 1.0)
    assert float((want - mean).abs().max()) > 0.05


@pytest.mark.parametrize("H,Hk,n", [(2, 2, 1), (2, 2, 4), (8, 2, 4)])
def test_queries_and_scales_at_opposite_ends(H, Hk, n):
    """Scores far above 1 and far below it: one key has all the weight, or all have the same."""
    lens = [1000, 70]
    q, cache, table, sl = _case(64, H, Hk, 16, lens, n, seed=32)
    for f, scale in ((1e-38, 1e-30), (1e-30, 1e-37), (1e-38, 1.0)):
        x = (q.float() * f).to(torch.bfloat16)
        _close(_run(x, cache, table, sl, scale=scale), *_exact(x, cache, table, lens, [n] * 2, scale))
    # a key 10 % above all others, in every head
    k, v, s = cache
    s2 = torch.nan_to_num(s.float(), nan=0.5)
    g = torch.Generator().manual_seed(33)
    s2[..., 0] = 0
    s2[..., 1] = (torch.rand(s2.shape[:3], generator=g).to(DEV) + 1)[..., None]
    for b, at in ((0, 700), (1, 40)):
        s2[int(table[b, at // 16]), :, at % 16, :, 1] = 2.25
    cache = (k, v, s2.to(torch.bfloat16))
    for f, scale in ((1e30, 1e4), (1e36, 0.1), (1e-2, 1e37), (1.0, 1e36)):
        x = torch.full_like(q, f)
        _close(_run(x, cache, table, sl, scale=scale), *_exact(x, cache, table, lens, [n] * 2, scale))

# ------------------------------------------------------------------ the longest sequence
@pytest.mark.parametrize("H,n", [(1, 1), (2, 2), (2, 4)])
def test_the_longest_sequence(H, n):
    """2^31 - 1 keys, of a few pages many times over: the place behind the last one stays hidden. Every
    value is 1 and so is their mean, to fp32 sums of 2^31 terms over 2^16 threads (2^15 a thread, each addition
    within 2^-24) and the result's rounding."""
    page, longest = 256, (1 << 31) - 1
    g = torch.Generator().manual_seed(41)
    k = torch.randint(0, 256, (3, 1, page, 32), generator=g, dtype=torch.uint8).to(DEV)
    v = torch.zeros_like(k)
    s = torch.zeros(3, 1, page, 1, 4, dtype=torch.bfloat16, device=DEV)
    s[..., 3] = 1.0
    s[2, :, -1, :, 1], s[2, :, -1, :, 3] = 50.0, 1000.0      # behind the end, with all the weight
    table = torch.arange((1 << 31) // page, device=DEV, dtype=torch.int32)[None] % 2
    table[0, -1] = 2
    q = torch.ones(1, n, H, 64, dtype=torch.bfloat16, device=DEV)
    sl = torch.tensor([longest], dtype=torch.int32, device=DEV)
    got = _run(q, (k, v, s), table, sl, max_len=longest)
    assert float((got.double() - 1).abs().max()) <= 2.0 ** -7, got.flatten()[:4]
