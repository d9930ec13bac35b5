"""GPU tests of the serving operators at their edges: calls without keys, values that
are not finite, scales and lengths at the ends of their ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("B,H,Hk,hd", [(64, 16, 16, 64), (40, 32, 32, 128), (300, 40, 1, 128), (2, 4, 2, 64)])
@pytest.mark.parametrize("pages", [0, 3])
def test_decode_without_keys(B, H, Hk, hd, pages):
    """max_len 0: zeros for sequences without keys, NaN for those that claim some, as
    many lists as there are."""
    from naylis_b200 import attention
    q = _rand(1, B, H, hd)
    kp, vp = _rand(2, 3, Hk, 16, hd), _rand(3, 3, Hk, 16, hd)
    table = torch.zeros(B, pages, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    lens[B // 2] = -4
    assert bool((attention.decode_attention(q, kp, vp, table, lens, max_len=0) == 0).all())
    lens[0], lens[B - 1] = 1, 1 << 30
    out = attention.decode_attention(q, kp, vp, table, lens, max_len=0)
    assert bool(torch.isnan(out[[0, B - 1]]).all()) and bool((out[1:B - 1] == 0).all())



def _paged(seed, lens, Hk, page, hd):
    need = [-(-n // page) for n in lens]
    kp, vp = _rand(seed, sum(need) + 1, Hk, page, hd), _rand(seed + 1, sum(need) + 1, Hk, page, hd)
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return kp, vp, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


def _place(table, b, j, page):
    return int(table[b, j // page]), j % page


# lists that fit as clusters, and more than that: spans, one of them over many CTAs
BATCHES = [([1, 40, 700, 2], 64, 4, 2), ([1, 40, 700, 2], 128, 2, 2), ([5000] + [33] * 199, 64, 4, 4),
           ([5000] + [33] * 199, 128, 20, 2)]


@pytest.mark.parametrize("lens,hd,H,Hk", BATCHES)
def test_decode_scores_of_minus_infinity(lens, hd, H, Hk):
    """A sequence whose scores are all -inf has no softmax: NaN, as torch's; one key with a
    finite score takes all the weight."""
    from naylis_b200 import attention
    page = 16
    kp, vp, table, sl = _paged(4, lens, Hk, page, hd)
    q = _rand(6, len(lens), H, hd)
    q[..., 0] = 1.0
    kp[..., 0] = float("-inf")
    alone = [0, 17]      # of sequences 0 and 1
    for b, j in enumerate(alone):
        if j < lens[b]:
            at, off = _place(table, b, j, page)
            kp[at, :, off, 0] = 0.5
    out = attention.decode_attention(q, kp, vp, table, sl)
    for b, j in enumerate(alone):
        at, off = _place(table, b, j, page)
        want = vp[at, :, off].repeat_interleave(H // Hk, 0)
        assert torch.equal(out[b], want)
    assert bool(torch.isnan(out[2:]).all())


@pytest.mark.parametrize("lens,hd,H,Hk", BATCHES)
def test_decode_infinite_values(lens, hd, H, Hk):
    """An infinite value that a sequence sees makes its column infinite, of its sign; two
    of different signs NaN; the other columns, heads and sequences keep their results."""
    from naylis_b200 import attention
    page, inf = 16, float("inf")
    kp, vp, table, sl = _paged(8, lens, Hk, page, hd)
    q = _rand(10, len(lens), H, hd)
    clean = attention.decode_attention(q, kp, vp, table, sl)
    a, ao = _place(table, 1, 5, page)
    vp[a, 0, ao, 3], vp[a, Hk - 1, ao, 7] = inf, -inf
    a, ao = _place(table, 1, 21, page)
    vp[a, 0, ao, 3], vp[a, 0, ao, 4] = -inf, inf
    G = H // Hk
    want = clean.clone()
    want[1, :G, 3] = float("nan")
    want[1, :G, 4] = inf
    want[1, H - G:, 7] = -inf
    out = attention.decode_attention(q, kp, vp, table, sl)
    special = ~torch.isfinite(want)
    assert torch.equal(out[special].nan_to_num(nan=5.0), want[special].nan_to_num(nan=5.0))
    assert torch.equal(out[~special], clean[~special])


@pytest.mark.parametrize("lens,hd,H,Hk", BATCHES)
def test_decode_is_rounded_once(lens, hd, H, Hk):
    """The weights' two terms hold them to 2^-16: of the output's half ulp (2^-8 of it),
    2^-12 of sum p |v| is left for them, the exponential and the sums."""
    from naylis_b200 import attention
    page = 16
    kp, vp, table, sl = _paged(12, lens, Hk, page, hd)
    q = _rand(14, len(lens), H, hd, scale=2.0)
    out = attention.decode_attention(q, kp, vp, table, sl).double()
    for b in (0, 1, 2, 3, len(lens) - 1):
        ids = table[b, :-(-lens[b] // page)].long()
        k, v = (t[ids].transpose(1, 2).reshape(-1, Hk, hd)[:lens[b]].double().repeat_interleave(H // Hk, 1)
                for t in (kp, vp))
        p = torch.softmax(torch.einsum("hd,jhd->hj", q[b].double(), k) * hd ** -0.5, -1)
        want, A = torch.einsum("hj,jhd->hd", p, v), torch.einsum("hj,jhd->hd", p, v.abs())
        assert bool(((out[b] - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * A).all())
