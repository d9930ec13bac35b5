"""GPU tests of token_logprobs away from centred logits: large offsets, small
temperatures and masks, against the definition in 64 bits.

Tolerances, u = 2^-24, y_j = (x_j - max) / T, p the probabilities:
  e^y_j      its argument takes five roundings (1 / T, log2 e, their product, the
             difference, the last product), the exponential is within 2^-22 = 4 u:
             relative 5 u |y_j| + 4 u <= E_j = 8 u (1 + |y_j|)
  ln Z       e_z = n u + sum p_j E_j, n = V / 32 + 64 additions to a sum
  logprob    e_z + 8 u (1 + |logprob| + |y_t|)
  entropy    ln Z - sum p y: e_z (1 + S) + (n + 16) u S + sum p_j |y_j| E_j + 8 u (1 + H),
             S = sum p_j |y_j|
  gradient   -p_j (G + h (y_j - ln Z + H)) and the single elements' terms, over T: p_j within e_z + E_j,
             the bracket within 16 u of its terms' magnitudes and |h| (e_H + e_z), the single terms within 8 u;
             half an ulp of a bf16 result on top (2^-8 of it). Probabilities below 2^-126 may be 0.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24


def _check(x, top, T, seed=0, backward=True):
    from naylis_b200 import scoring
    R, V = x.shape
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (R,), generator=g).to(DEV)
    best = x.float().argmax(-1)
    t[::2] = best[::2]
    xg = x.clone().requires_grad_(backward)
    r = scoring.token_logprobs(xg, t, top_k=top, temperature=T)
    x64 = x.double()
    y = (x64 - x64.amax(-1, keepdim=True)) / T
    lz = torch.logsumexp(y, -1, keepdim=True)
    lp = y - lz
    p = lp.exp()
    dead = p == 0
    ay = torch.where(dead, 0.0, y.abs())
    H = -torch.where(dead, 0.0, p * lp).sum(-1, keepdim=True)
    n = V / 32 + 64
    E = 8 * U * (1 + ay)
    ez = n * U + (p * E).sum(-1, keepdim=True)
    S = (p * ay).sum(-1, keepdim=True)
    eH = ez * (1 + S) + (n + 16) * U * S + (p * ay * E).sum(-1, keepdim=True) + 8 * U * (1 + H)

    def close(got, want, ays):
        want32 = want.float()                      # what fp32 cannot hold is infinite there
        same = got == want32
        return bool((same | ((got.double() - want).abs() <= ez + 8 * U * (1 + want.abs() + ays))).all())

    assert close(r.logprob[:, None], lp.gather(1, t[:, None]), ay.gather(1, t[:, None]))
    assert bool(((r.entropy[:, None].double() - H).abs() <= eH).all())
    if top:
        idx = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(r.top_idx, idx)
        assert close(r.top_logprob, lp.gather(1, idx), ay.gather(1, idx))
    if not backward:
        return
    gl, h = (torch.randn(R, 1, generator=g).to(DEV) for _ in range(2))
    a = torch.randn(R, max(top, 1), generator=g).to(DEV) if top else None
    outs, gs = [r.logprob, r.entropy], [gl[:, 0], h[:, 0]]
    if top:
        outs.append(r.top_logprob)
        gs.append(a)
    d, = torch.autograd.grad(outs, xg, gs)
    gl, h = gl.double(), h.double()
    pick = torch.zeros_like(p).scatter_add_(1, t[:, None], gl)
    if top:
        pick.scatter_add_(1, idx, a.double())
    sumg = gl.abs() + (a.double().abs().sum(-1, keepdim=True) if top else 0)
    inner = torch.where(dead, 0.0, pick.sum(-1, keepdim=True) + h * (lp + H))
    want = (pick - p * inner) / T
    size = sumg + h.abs() * (ay + lz.abs() + H)
    tol = (p * (size * (ez + E + 16 * U) + h.abs() * (eH + ez)) + 8 * U * pick.abs()) / T + 4 * U * want.abs()
    if d.dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    assert bool(((d.double() - want).abs() <= tol + 2.0 ** -100 / T).all())


# bf16 and fp32 rows of these lengths go to a warp, 128 threads and 512 threads
LENGTHS = [(torch.bfloat16, 1001), (torch.bfloat16, 6001), (torch.bfloat16, 32003), (torch.float32, 999),
           (torch.float32, 3001), (torch.float32, 9001)]


def _base(seed, R, V, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * 3).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype,V", LENGTHS)
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_offsets(dtype, V, T):
    """Logits far from 0: what counts is their distance from the maximum."""
    off = torch.tensor([0.0, 30.0, -1e3, 1e4, 1e6, -1e6, -1e10, 1e20], device=DEV)
    x = (_base(V, len(off), V, torch.float32) + off[:, None]).to(dtype)
    _check(x, 5, T)


@pytest.mark.parametrize("dtype,V", LENGTHS)
@pytest.mark.parametrize("T", [1e-6, 1e-3, 0.01, 1e3, 1e6])
def test_temperatures(dtype, V, T):
    x = _base(V + 1, 4, V, dtype)
    x[1] += 100
    _check(x, 5, T)


def _patterns(base, fill):
    """Rows in which `fill` stands in places that a mask leaves it in: all but a few, all
    but one, the whole row, single elements at its ends, its halves, next to -inf."""
    x = base[:10].clone()
    V = x.shape[1]
    keep = torch.randperm(V, generator=torch.Generator().manual_seed(V))[:10].to(DEV)
    x[0] = fill
    x[0, keep] = base[0, keep]
    x[1] = fill
    x[2, 0] = fill
    x[3, -1] = fill
    x[4, :V // 2] = fill
    x[5, V // 2:] = fill
    x[6, :-1] = fill
    x[7, 1:] = fill
    x[8] = fill
    x[8, ::3] = float("-inf")
    x[9, ::2] = fill
    return x


@pytest.mark.parametrize("dtype,V", LENGTHS)
@pytest.mark.parametrize("fill", [-1e4, -65504.0, -1e9, -1e10, -1e12, -1e20])
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_finite_masks(dtype, V, fill, T):
    _check(_patterns(_base(V + 2, 10, V, dtype), fill), 20, T)


@pytest.mark.parametrize("dtype,V", LENGTHS)
@pytest.mark.parametrize("fill", [-1e30, -3e38, "lowest", -5e29, 1e30, "greatest"])
@pytest.mark.parametrize("T", [1.0, 0.7, 1e-6, 1e6])
def test_masks_of_the_lowest_value(dtype, V, fill, T):
    """Down to the type's lowest value, and up to its greatest."""
    ends = {"lowest": torch.finfo(dtype).min, "greatest": torch.finfo(dtype).max}
    _check(_patterns(_base(V + 3, 10, V, dtype), ends.get(fill, fill)), 20, T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_short_rows_of_masks(dtype):
    """Rows of one to nine elements, none of whose threads has a whole vector."""
    low = torch.finfo(dtype).min
    for V in range(1, 10):
        x = _base(V, 12, V, dtype)
        x[:6] = low
        x[1, V // 2] = float("-inf") if V > 1 else low
        x[2, 0] = 2.0
        x[3, -1] = -1e30
        x[4, V // 2] = torch.finfo(dtype).max
        x[7, 0] = low
        x[8, -1] = low
        _check(x, min(V, 3), 1.0)


@pytest.mark.parametrize("dtype,V", LENGTHS)
@pytest.mark.parametrize("T,weight", [(1e-6, 1e4), (1e-3, 1e9), (1.0, 1e10)])
def test_gradient_of_masked_logits_is_zero(dtype, V, T, weight):
    """However much the entropy's gradient weighs: 0 where the probability is, and
    finite elsewhere (two equal logits share the row: p = 1/2, H = ln 2, no gradient)."""
    from naylis_b200 import scoring
    for fill in (float("-inf"), torch.finfo(dtype).min, -1e30):
        x = torch.full((2, V), fill, dtype=dtype, device=DEV)
        x[:, 5], x[:, V - 1] = 1.5, 1.5
        x.requires_grad_(True)
        r = scoring.token_logprobs(x, torch.tensor([5, 7], device=DEV), temperature=T)
        d, = torch.autograd.grad(r.entropy, x, torch.full((2,), weight, device=DEV))
        gone = torch.ones(V, dtype=torch.bool, device=DEV)
        gone[[5, V - 1]] = False
        assert bool((d[:, gone] == 0).all())
        # ln p + H is 0 within 32 u of ln 2: e_z and the roundings of its terms
        assert bool((d.double().abs() <= weight / T * (V / 32 + 64 + 32) * U).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_target_outside_spoils_its_logprob_alone(dtype):
    """The entropy's and the alternatives' gradients do not depend on the target."""
    from naylis_b200 import scoring
    V, top = 300, 4
    x = _base(3, 4, V, dtype).requires_grad_(True)
    outside = torch.tensor([V, -1, 3, 1 << 40], device=DEV)
    inside = torch.tensor([0, 1, 3, 7], device=DEV)
    bad = torch.tensor([True, True, False, True], device=DEV)
    g, a = torch.randn(4, device=DEV), torch.randn(4, top, device=DEV)

    def gradient(t, which):
        r = scoring.token_logprobs(x, t, top_k=top)
        return torch.autograd.grad([r[i] for i in which], x, [g if i < 2 else a for i in which])[0]

    for which in ((1,), (3,), (1, 3)):
        assert torch.equal(gradient(outside, which), gradient(inside, which))
    for which in ((0,), (0, 1)):
        d = gradient(outside, which)
        assert bool(torch.isnan(d[bad]).all()) and torch.equal(d[~bad], gradient(inside, which)[~bad])
