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


def _prompt_want(q, k, v, lens, scale):
    """Per row and column: what the values that a row sees make of it (NaN, or infinities
    of one sign, there decide; else the sum), in 64 bits, with sum p |v|."""
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    outs, sizes, o = [], [], 0
    for n in lens:
        qs, ks, vs = (t[o:o + n].double().transpose(0, 1) for t in (q, k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)))
        see = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        p = torch.softmax((qs @ ks.transpose(1, 2) * scale).masked_fill(~see, float("-inf")), -1)
        plain = torch.where(torch.isfinite(vs), vs, 0.0)
        out, size = p @ plain, p @ plain.abs()
        seen = lambda hit: torch.cummax(hit.int(), 1)[0].bool()
        nan, up, down = seen(torch.isnan(vs)), seen(vs == float("inf")), seen(vs == float("-inf"))
        out[up] = float("inf")
        out[down] = float("-inf")
        out[nan | (up & down)] = float("nan")
        out[torch.isnan(p.sum(-1))] = float("nan")
        outs.append(out.transpose(0, 1))
        sizes.append(size.transpose(0, 1))
        o += n
    return torch.cat(outs), torch.cat(sizes)


def _prompt_check(q, k, v, lens):
    from naylis_b200 import attention
    scale = 0.25 * q.shape[2] ** -0.5
    plan = attention.PromptPlan(lens, device=DEV)
    out = attention.prompt_attention(q, k, v, plan, scale=scale).double()
    plan.check()
    want, size = _prompt_want(q, k, v, lens, scale)
    special = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out[special].nan_to_num(nan=5.0), want[special].nan_to_num(nan=5.0))
    tol = 2.0 ** -7 + 2.0 ** -12      # weights and output rounded to bf16, the exponential
    assert bool(((out - want).abs()[~special] <= tol * size[~special] + 2.0 ** -40).all())


@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (64, 4, 2), (128, 4, 2), (128, 3, 1)])
def test_prompt_values_that_are_not_finite(hd, H, Hk):
    """Each row and column by itself: hidden values leave no trace, seen ones decide, and a
    row without a softmax is NaN whatever its values are."""
    lens, inf, nan = [300, 140, 257], float("inf"), float("nan")
    q, k, v = (_rand(20 + i, sum(lens), h, hd) for i, h in enumerate((H, Hk, Hk)))
    last = Hk - 1
    v[200, 0, 3], v[210, 0, 3] = nan, inf
    v[90, 0, 4], v[220, 0, 4] = -inf, inf
    v[299, last, 5], v[150, last, 5] = inf, inf
    v[130, last, 6] = -inf
    v[299, 0], v[300, 0] = nan, inf              # the first sequence's last row, the second's first
    k[500, 0, 1] = nan
    v[520, 0, 7], v[440 + 256, 0, 7] = inf, nan
    _prompt_check(q, k, v, lens)


@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (128, 4, 2), (128, 3, 3)])
@pytest.mark.parametrize("q_lens,k_lens", [([64, 200, 5], [10, 455, 3]), ([300, 130], [172, 258]), ([1, 33, 129], [300, 400, 129])])
def test_prompt_hidden_values_behind_a_prefix(hd, H, Hk, q_lens, k_lens):
    """More keys than queries, and fewer (rows without one stay 0): values of the last key
    of each sequence, and of one in its middle, are NaN or infinite."""
    from naylis_b200 import attention
    q, k, v = (_rand(60 + i, n, h, hd) for i, (n, h) in enumerate(
        ((sum(q_lens), H), (sum(k_lens), Hk), (sum(k_lens), Hk))))
    end = 0
    for m in k_lens:
        v[end + m // 2, 0, 1], v[end + m // 2, Hk - 1, 2] = float("inf"), float("nan")
        end += m
        v[end - 1, :, 3], v[end - 1, 0, 4] = float("nan"), float("-inf")
    scale = 0.25 * hd ** -0.5
    plan = attention.PromptPlan(q_lens, k_lens, device=DEV)
    out = attention.prompt_attention(q, k, v, plan, scale=scale).double()
    plan.check()
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        for r in range(n):
            seen, got = m - n + r + 1, out[a + r]
            if seen <= 0:
                assert bool((got == 0).all())
                continue
            ks, vs = (t[b:b + seen].double().repeat_interleave(H // Hk, 1) for t in (k, v))
            p = torch.softmax(torch.einsum("hd,jhd->hj", q[a + r].double(), ks) * scale, -1)
            plain = torch.where(torch.isfinite(vs), vs, 0.0)
            want, size = torch.einsum("hj,jhd->hd", p, plain), torch.einsum("hj,jhd->hd", p, plain.abs())
            want[(vs == float("inf")).any(0)] = float("inf")
            want[(vs == float("-inf")).any(0)] = float("-inf")
            want[torch.isnan(vs).any(0)] = float("nan")
            special = ~torch.isfinite(want)
            assert torch.equal(got[special].nan_to_num(nan=5.0), want[special].nan_to_num(nan=5.0))
            tol = 2.0 ** -7 + 2.0 ** -12
            assert bool(((got - want).abs()[~special] <= tol * size[~special] + 2.0 ** -40).all())
        a, b = a + n, b + m


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fill", ["nan", "inf", "one", "both"])
def test_prompt_values_of_a_diverged_model(hd, fill):
    """Values that are NaN, infinite of one sign or of both throughout, or for one token."""
    lens, H, Hk = [513, 200], 4, 2
    q, k, v = (_rand(30 + i, sum(lens), h, hd) for i, h in enumerate((H, Hk, Hk)))
    if fill == "one":
        v[500] = float("nan")
    elif fill == "both":
        v[:] = torch.where(v > 0, float("inf"), float("-inf")).to(v.dtype)
    else:
        v[:] = float(fill)
    _prompt_check(q, k, v, lens)


@pytest.mark.parametrize("hd,H,Hk", [(64, 16, 16), (128, 16, 4)])
def test_prompt_of_nan_values_takes_no_longer(hd, H, Hk):
    """A diverged model's values leave nothing to compute again: the call stays within 4
    times an ordinary one's (the rows are looked at once more: for 4096 rows of 16 heads
    some 100 us behind the 100 to 150 of the call)."""
    from naylis_b200 import attention
    n = 4096
    q, k, v = (_rand(40 + i, n, h, hd) for i, h in enumerate((H, Hk, Hk)))
    plan = attention.PromptPlan([n], device=DEV)

    def least(values):
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                attention.prompt_attention(q, k, values, plan)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    plain = least(v)
    assert least(torch.full_like(v, float("nan"))) <= 4 * plain


def test_a_plan_outlives_its_use_on_another_stream():
    """A plan's list, made on one stream and read on another, is not given to a new tensor
    while the other stream's work is pending. (Nothing reads the list here.)"""
    from naylis_b200 import attention
    plan = attention.PromptPlan([300, 20], device=DEV)
    buffer = plan.list_for(4, 2)
    at, size = buffer.data_ptr(), buffer.numel()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)      # about 0.1 s
        assert plan.list_for(4, 2) is buffer
    del plan, buffer
    others = [torch.empty(size, dtype=torch.uint8, device=DEV) for _ in range(4)]
    pending = not side.query()
    assert all(t.data_ptr() != at for t in others) and pending
    side.synchronize()


def test_derivatives_are_refused_not_dropped():
    """Forward-mode tangents, and tables that require grad, as any input that does."""
    from torch.autograd import forward_ad

    from naylis_b200 import attention, scoring
    hd, H, Hk, T = 64, 2, 1, 3
    qkv = _rand(1, T, (H + 2 * Hk) * hd)
    kp, vp = _rand(2, 1, Hk, 16, hd), _rand(3, 1, Hk, 16, hd)
    cos, sin = torch.ones(T, hd, device=DEV), torch.zeros(T, hd, device=DEV)
    at = torch.arange(T, device=DEV)
    q, k = _rand(4, T, H, hd), _rand(5, T, Hk, hd)
    plan = attention.PromptPlan([T], device=DEV)
    table, lens = torch.zeros(T, 1, dtype=torch.int32, device=DEV), torch.ones(T, dtype=torch.int32, device=DEV)
    logits, target = torch.randn(T, 50, device=DEV), at
    calls = [(lambda x: attention.rope_append(x, cos, sin, at, kp, vp, at, n_heads=H), qkv),
             (lambda x: attention.rope_append(qkv, x, sin, at, kp, vp, at, n_heads=H), cos),
             (lambda x: attention.rope_append(qkv, cos, x, at, kp, vp, at, n_heads=H), sin),
             (lambda x: attention.prompt_attention(x, k, k, plan), q),
             (lambda x: attention.decode_attention(x, kp, vp, table, lens), q)]
    for call, x in calls:
        call(x)
        with pytest.raises(RuntimeError, match="forward only"):
            call(x.clone().requires_grad_(True))
        with torch.no_grad():
            call(x.clone().requires_grad_(True))
    calls.append((lambda x: scoring.token_logprobs(x, target), logits))
    with forward_ad.dual_level():
        for call, x in calls:
            call(x)
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
