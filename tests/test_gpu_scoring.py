"""GPU tests of token_logprobs (naylis_b200/scoring.py) against its definition in
64 bits, its gradient against the formula's and against differences.

Tolerances, from fp32 arithmetic with unit roundoff u = 2^-24: a row's sum over V
terms in partial sums of at most V / 32 terms each is within n u of its
magnitude, n = V / 32 + 64; an exponential of y is within 4 u (1 + |y|), the
argument's own roundings among them. With S = sum_j p_j |y_j| + 1:
  Z, ln Z        e_z = n u + 4 u S                 (relative / absolute)
  logprob        e_z + 4 u (|logprob| + |y|)
  entropy        (e_z + n u + 4 u S) S + 4 u (1 + H)
  p_j            relative e_p = e_z + 4 u (1 + |y_j|)
and the gradient's terms by these, plus half an ulp of its dtype.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24


def _logits(seed, R, V, dtype, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * scale).to(dtype).to(DEV)


def _exact(x, t, top, T, ignore=-100):
    x64 = x.detach().double()
    y = x64 / T
    lp = torch.log_softmax(y, -1)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    live = t != ignore
    inside = live & (t >= 0) & (t < x.shape[1])
    one = lp.gather(1, torch.where(inside, t, 0)[:, None])[:, 0]
    one = torch.where(inside, one, torch.where(live, float("nan"), 0.0))
    # value descending, index ascending; -0 ties with 0
    idx = torch.sort(x.detach().float() + 0.0, dim=-1, descending=True, stable=True)[1][:, :top]
    return lp, p, H, one, idx, lp.gather(1, idx)


def _bounds(lp, p, x, T):
    V = x.shape[1]
    n = V / 32 + 64
    y = (x.detach().double() - x.detach().double().amax(-1, keepdim=True)) / T
    ay = torch.where(p > 0, y.abs(), 0.0)
    S = (p * ay).sum(-1) + 1
    ez = n * U + 4 * U * S
    return ay, S, ez, n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,top,T", [(1, 1, 1, 1.0), (3, 2, 2, 0.7), (5, 33, 32, 1.0), (2, 1000, 8, 1.3),
                                       (7, 4099, 20, 1.0), (3, 32000, 5, 1.0), (300, 777, 1, 1.0), (2, 70001, 32, 0.5)])
def test_forward(dtype, R, V, top, T):
    from naylis_b200 import scoring
    x = _logits(R + V, R, V, dtype)
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(1)).to(DEV)
    if R > 1:
        t[0] = -100
    r = scoring.token_logprobs(x, t, top_k=top, temperature=T)
    lp, p, H, one, idx, top_lp = _exact(x, t, top, T)
    ay, S, ez, n = _bounds(lp, p, x, T)
    assert torch.equal(r.top_idx, idx)
    ty = ay.gather(1, t.clamp_min(0)[:, None])[:, 0]
    assert bool(((r.logprob.double() - one).abs() <= ez + 4 * U * (one.abs() + ty)).all())
    assert bool(((r.top_logprob.double() - top_lp).abs()
                 <= ez[:, None] + 4 * U * (top_lp.abs() + ay.gather(1, idx))).all())
    assert bool(((r.entropy.double() - H).abs() <= (ez + n * U + 4 * U * S) * S + 4 * U * (1 + H)).all())
    plain = scoring.token_logprobs(x, t, temperature=T)
    assert plain.top_idx is None and plain.top_logprob is None
    assert torch.equal(plain.logprob, r.logprob) and torch.equal(plain.entropy, r.entropy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [64, 5000, 32000])
def test_ties_go_to_the_lowest_index(dtype, V):
    """Equal logits everywhere, a few levels, signed zeros, and a maximum at the end."""
    from naylis_b200 import scoring
    top = 32
    g = torch.Generator().manual_seed(3)
    rows = [torch.zeros(V), torch.full((V,), -2.5), torch.randint(0, 3, (V,), generator=g).float(),
            torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), torch.arange(V).float() // (V // 8)]
    rows.append(rows[2].clone())
    rows[-1][-1] = 9.0
    x = torch.stack(rows).to(dtype).to(DEV)
    t = torch.zeros(len(rows), dtype=torch.int64, device=DEV)
    r = scoring.token_logprobs(x, t, top_k=top)
    assert torch.equal(r.top_idx, _exact(x, t, top, 1.0)[4])


def test_masked_and_broken_rows():
    """-inf logits have probability 0; a row with NaN or +inf, or all -inf, is NaN;
    targets: ignored 0, outside the vocabulary NaN, masked -inf."""
    from naylis_b200 import scoring
    V, inf, nan = 300, float("inf"), float("nan")
    x = _logits(5, 8, V, torch.float32)
    x[0, 10:] = -inf
    x[1, :] = -inf
    x[2, 7] = nan
    x[3, 9] = inf
    x[4, 1:] = -inf
    x[5, 4] = torch.finfo(torch.float32).min
    t = torch.tensor([3, 3, 3, 3, 0, 4, 400, 20], device=DEV)
    x[7, 20] = -inf
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype).requires_grad_(True)
        r = scoring.token_logprobs(xd, t, top_k=12)
        y = torch.log_softmax(xd.detach().double(), -1)
        p = y.exp()
        H = -torch.where(p > 0, p * y, 0.0).sum(-1)
        for i in (0, 4, 5, 7):
            assert abs(float(r.entropy[i].double() - H[i])) <= 1e-5
            ref = y[i, t[i]]
            got = r.logprob[i].double()
            assert bool(got == ref) or abs(float(got - ref)) <= 1e-6 * max(1.0, abs(float(ref)))
        assert bool((r.top_logprob[0, 10:] == -inf).all()) and r.top_idx[0, 10:].tolist() == [10, 11]
        assert r.top_idx[4].tolist() == list(range(12)) and r.top_idx[1].tolist() == list(range(12))
        assert int(r.top_idx[2, 0]) == 7 and int(r.top_idx[3, 0]) == 9
        for i in (1, 2, 3):
            assert bool(torch.isnan(r.logprob[i])) and bool(torch.isnan(r.entropy[i]))
        assert bool(torch.isnan(r.logprob[6])) and abs(float(r.entropy[6].double() - H[6])) <= 1e-5
        d, = torch.autograd.grad([r.logprob, r.entropy], xd, [torch.ones(8, device=DEV)] * 2)
        assert bool((d[0, 10:] == 0).all()) and bool(torch.isfinite(d[0].float()).all())
        assert bool(torch.isfinite(d[[4, 5, 7]].float()).all())
        assert bool(torch.isnan(d[[1, 2, 3, 6]].float()).all(1).all())


def _grad_exact(x, t, top, T, g, h, a):
    lp, p, H, _, idx, _ = _exact(x, t, top, T)
    live = t != -100
    g = g.double() * live
    pick = torch.zeros_like(p).scatter_add_(1, t.clamp_min(0)[:, None], g[:, None])
    if top:
        pick.scatter_add_(1, idx, a.double())
    G = pick.sum(-1, keepdim=True)
    d = (pick - p * (G + h.double()[:, None] * (lp + H[:, None]))) / T
    return d, lp, p, H, pick.abs(), g.abs()[:, None] + (a.double().abs().sum(-1, keepdim=True) if top else 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,top,T", [(1, 1, 0, 1.0), (4, 33, 3, 0.7), (3, 4099, 20, 1.0), (2, 32000, 0, 1.3)])
def test_gradient_against_the_formula(dtype, R, V, top, T):
    from naylis_b200 import scoring
    x = _logits(R * V, R, V, dtype).requires_grad_(True)
    gen = torch.Generator().manual_seed(2)
    t = torch.randint(0, V, (R,), generator=gen).to(DEV)
    if R > 2:
        t[1] = -100
    g, h = (torch.randn(R, generator=gen).to(DEV) for _ in range(2))
    a = torch.randn(R, max(top, 1), generator=gen).to(DEV)
    r = scoring.token_logprobs(x, t, top_k=top, temperature=T)
    outs, gs = [r.logprob, r.entropy], [g, h]
    if top:
        outs.append(r.top_logprob)
        gs.append(a)
    d, = torch.autograd.grad(outs, x, gs)
    assert d.dtype == dtype and d.shape == x.shape
    want, lp, p, H, pick, sumg = _grad_exact(x, t, top, T, g, h, a)
    ay, S, ez, n = _bounds(lp, p, x, T)
    ep = ez[:, None] + 4 * U * (1 + ay)
    alp = torch.where(p > 0, lp.abs(), 0.0)
    inner = sumg + h.double().abs()[:, None] * (alp + H[:, None])
    eH = ((ez + n * U + 4 * U * S) * S + 4 * U * (1 + H))[:, None]
    e_inner = 8 * U * inner + 32 * U * sumg + h.double().abs()[:, None] * (eH + ep * 1.0 + 4 * U * (alp + ay))
    tol = (p * (inner * (ep + 4 * U) + e_inner) + 4 * U * pick) / T + 4 * U * want.abs()
    if dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()      # half an ulp of 8 significant bits
    assert bool(((d.double() - want).abs() <= tol + 2.0 ** -130).all())


def test_each_gradient_alone_and_none():
    """Only one of the outputs used, and an output used twice."""
    from naylis_b200 import scoring
    R, V, top = 3, 50, 4
    x = _logits(11, R, V, torch.float32).requires_grad_(True)
    t = torch.tensor([1, 49, -100], device=DEV)
    zero = torch.zeros(R, device=DEV)
    g = torch.randn(R, device=DEV)
    a = torch.randn(R, top, device=DEV)
    for outs, gs, args in [((0,), (g,), (g, zero, 0 * a)), ((1,), (g,), (zero, g, 0 * a)), ((3,), (a,), (zero, zero, a)),
                           ((0, 3), (g, a), (g, zero, a))]:
        r = scoring.token_logprobs(x, t, top_k=top)
        d, = torch.autograd.grad([r[i] for i in outs], x, list(gs))
        want = _grad_exact(x, t, top, 1.0, *args)[0]
        assert float((d.double() - want).abs().max()) <= 1e-5
    # a broadcast upstream gradient (a sum) and an expanded one
    scoring.token_logprobs(x, t, top_k=top).entropy.sum().backward()
    want = _grad_exact(x, t, top, 1.0, zero, torch.ones_like(g), 0 * a)[0]
    assert float((x.grad.double() - want).abs().max()) <= 1e-5


def test_gradient_against_differences():
    """Central differences of the kernel's own forward, step s = 2^-5 (exact to add),
    the alternatives held at their indices (their order may change within a step):
    truncation s^2/6 of the third derivative, at most 3 (|g| + 4 |h| (1 + H) + ...)
    <= 40 here for unit weights, so 6.6e-3; rounding (2 x 3e-5) / (2 s) = 1e-3."""
    from naylis_b200 import scoring
    V, top = 9, 3
    x = (_logits(13, 1, V, torch.float32, scale=1.0) * 64).round() / 64
    x = x + torch.arange(V, device=DEV) * 0.25
    t = torch.tensor([4], device=DEV)
    g, h, a = torch.tensor([0.8]), torch.tensor([-0.6]), torch.tensor([[0.5, -0.7, 0.9]])

    xg = x.clone().requires_grad_(True)
    r = scoring.token_logprobs(xg, t, top_k=top)
    picked = torch.cat((t, r.top_idx[0]))

    def loss(z):
        q = scoring.token_logprobs(z.expand(1 + top, V), picked)
        weights = torch.cat((g, a[0])).double()
        return float((q.logprob.double().cpu() * weights).sum() + (q.entropy[:1].double().cpu() * h).sum())

    d, = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], xg, [g.to(DEV), h.to(DEV), a.to(DEV)])
    s = 2.0 ** -5
    for j in range(V):
        e = torch.zeros_like(x)
        e[0, j] = s
        num = (loss(x + e) - loss(x - e)) / (2 * s)
        assert abs(num - float(d[0, j])) <= 7.6e-3, (j, num, float(d[0, j]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_and_streams(dtype):
    """Rows that start off a 16-byte boundary, a pitch wider than the vocabulary, a
    transposed matrix (copied), another stream, a broadcast row."""
    from naylis_b200 import scoring
    R, V, top = 6, 1001, 7
    wide = _logits(17, R, V + 13, dtype)
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(4)).to(DEV)
    want = scoring.token_logprobs(wide[:, 3:3 + V].contiguous(), t, top_k=top)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = scoring.token_logprobs(wide[:, 3:3 + V], t, top_k=top)
    s.synchronize()
    turned = scoring.token_logprobs(wide[:, 3:3 + V].t().contiguous().t(), t.int(), top_k=top)
    for r in (got, turned):
        assert torch.equal(r.top_idx, want.top_idx)
        for x, y in ((r.logprob, want.logprob), (r.entropy, want.entropy), (r.top_logprob, want.top_logprob)):
            assert float((x - y).abs().max()) <= 2e-5      # sums in another order
    one = wide[:1, 3:3 + V].expand(R, V)
    b = scoring.token_logprobs(one, t, top_k=top)
    assert bool((b.top_idx == want.top_idx[0]).all())
    x = wide.clone().requires_grad_(True)
    r = scoring.token_logprobs(x[:, 3:3 + V], t, top_k=top)
    r.entropy.sum().backward()
    assert x.grad.shape == x.shape and bool((x.grad[:, :3] == 0).all()) and bool((x.grad[:, 3 + V:] == 0).all())
    assert torch.equal(scoring.token_logprobs(wide[:, 3:3 + V], t, top_k=top).logprob, got.logprob)


def test_large_logits_pass_32_bits():
    """Row offsets past 2^31 elements."""
    from naylis_b200 import scoring
    R, V = 33600, 64000
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    x[-1, 63999] = 12.0
    x[-2, 5] = 8.0
    t = torch.full((R,), 63999, device=DEV)
    x.requires_grad_(True)
    r = scoring.token_logprobs(x, t, top_k=2)
    assert r.top_idx[-2:].tolist() == [[5, 0], [63999, 0]]
    d, = torch.autograd.grad(r.logprob, x, torch.ones(R, device=DEV))
    want = torch.softmax(x.detach()[-2:].double(), -1)
    want = -want
    want[:, 63999] += 1
    assert float((d[-2:].double() - want).abs().max()) <= 2.0 ** -8


def test_refusals():
    from naylis_b200 import scoring
    x, t = _logits(1, 4, 20, torch.bfloat16), torch.zeros(4, dtype=torch.int64, device=DEV)
    assert scoring.token_logprobs(x[:0], t[:0], top_k=3).top_idx.shape == (0, 3)
    for args, kw in [((x.half(), t), {}), ((x.cpu(), t.cpu()), {}), ((x[0], t), {}), ((x, t[:3]), {}),
                     ((x, t.float()), {}), ((x, t), {"top_k": 21}), ((x, t), {"top_k": -1}), ((x, t), {"top_k": 33}),
                     ((x, t), {"temperature": 0.0}), ((x, t), {"temperature": float("nan")}),
                     ((x, t), {"temperature": float("inf")}), ((x[:, :0], t), {}), ((x, t.cpu()), {})]:
        with pytest.raises(RuntimeError):
            scoring.token_logprobs(*args, **kw)
