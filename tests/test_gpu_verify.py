"""GPU tests of scoring.verify_drafts against its definition in 64 bits: the tokens and
counts are whole numbers and have to be equal. (The kernel's sums and the definition's
differ by 1e-15 of them: a given number lands between the two with about that chance.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def _soft(x, T):
    y = x.double() / T
    if bool(torch.isnan(y).any()) or bool((y == INF).any()) or not bool((y > -INF).any()):
        return None
    return torch.softmax(y, -1)


def _want(logits, drafts, u, draft_logits, T, lens):
    """Row by row, on the CPU."""
    logits = logits.cpu()
    draft_logits = None if draft_logits is None else draft_logits.cpu()
    B, K = drafts.shape
    V = logits.shape[2]
    tokens, accepted = torch.full((B, K + 1), -1), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        n = K if lens is None else int(lens[b])
        if not 0 <= n <= K:
            continue
        j = 0
        while True:
            x = logits[b, j]
            if T == 0:
                nan = torch.isnan(x)
                best = -1 if bool(nan.any()) else int((x == x.max()).nonzero()[0])
                tokens[b, j] = best
                if j == n or best < 0 or int(drafts[b, j]) != best:
                    break
                j += 1
                continue
            p = _soft(x, T)
            if p is None:
                break
            if j == n:
                left = p
            else:
                d = int(drafts[b, j])
                inside = 0 <= d < V
                if draft_logits is None:
                    q = torch.zeros_like(p)
                    if inside:
                        q[d] = 1.0
                else:
                    q = _soft(draft_logits[b, j], T)
                    if q is None:
                        break
                if inside and float(u[b, j].double()) * float(q[d]) < float(p[d]):
                    tokens[b, j] = d
                    j += 1
                    continue
                left = torch.relu(p - q)
                if float(left.sum()) == 0.0:
                    left = p
            c = left.cumsum(0)
            at = int((c <= float(u[b, K].double()) * c[-1]).sum())
            tokens[b, j] = min(at, int((left > 0).nonzero()[-1]))
            break
        accepted[b] = j
    return tokens, accepted


def _make(seed, B, K, V, dtype, mode, T, noise=0.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, K + 1, V, generator=g) * 2).to(dtype)
    fav = torch.randint(0, V, (B, K + 1, 2), generator=g)
    logits.scatter_(2, fav, (8 + torch.rand(B, K + 1, 2, generator=g)).to(dtype))
    draft = (logits[:, :K].float() + noise * torch.randn(B, K, V, generator=g)).to(dtype)
    x = draft.float() / max(T, 1e-3)
    if mode != "greedy":
        x = x - torch.log(-torch.log(torch.rand(B, K, V, generator=g).clamp(1e-9, 1 - 1e-6)))
    drafts = x.argmax(-1) if K else torch.zeros(B, 0, dtype=torch.int64)
    u = torch.rand(B, K + 1, generator=g)
    return (logits.to(DEV), drafts.to(DEV), None if mode == "greedy" else u.to(DEV),
            draft.to(DEV) if mode == "sampled" else None)


def _check(logits, drafts, u, draft, T, lens=None):
    from naylis_b200 import scoring
    lt = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = scoring.verify_drafts(logits, drafts, u, draft_logits=draft, temperature=T, draft_lens=lt)
    want = _want(logits, drafts.cpu(), None if u is None else u.cpu(), draft, T, lens)
    assert torch.equal(got.tokens.cpu(), want[0]), (got.tokens.cpu(), want[0])
    assert torch.equal(got.accepted.cpu(), want[1])
    again = scoring.verify_drafts(logits, drafts, u, draft_logits=draft, temperature=T, draft_lens=lt)
    assert torch.equal(got.tokens, again.tokens) and torch.equal(got.accepted, again.accepted)
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mode,T", [("sampled", 1.0), ("sampled", 0.6), ("lookup", 1.0), ("lookup", 1.7), ("greedy", 0.0)])
@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (3, 1, 1), (5, 3, 2), (7, 8, 17), (40, 5, 257), (33, 4, 5003),
                                   (3, 32, 1000), (150, 3, 4096), (300, 2, 999), (9, 0, 3001)])
def test_against_the_definition(dtype, mode, T, B, K, V):
    seed = B * 1000 + K * 10 + V
    want = _check(*_make(seed, B, K, V, dtype, mode, T), T)
    if B >= 40 and mode == "sampled":      # the inputs reach every end
        assert len(set(want[1].tolist())) > 2
    lens = [(3 * i) % (K + 1) for i in range(B)]
    if B > 4:
        lens[1], lens[3] = -1, K + 1
    _check(*_make(seed + 1, B, K, V, dtype, mode, T), T, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [8, 1003, 32003])
def test_the_same_distribution_keeps_every_draft(dtype, V):
    logits, drafts, u, _ = _make(2, 8, 3, V, dtype, "sampled", 1.0)
    want = _check(logits, drafts, u, logits[:, :3].clone(), 1.0)
    assert want[1].tolist() == [3] * 8


def test_a_choice_on_the_border():
    """Numbers that 32-bit sums would put on the wrong side: u at p / q, and just beside."""
    V = 4099
    logits, drafts, u, draft = _make(4, 64, 2, V, torch.float32, "sampled", 1.0, noise=2.0)
    p, q = torch.softmax(logits[:, :2].double(), -1), torch.softmax(draft.double(), -1)
    r = (p.gather(2, drafts[..., None]) / q.gather(2, drafts[..., None]))[..., 0]
    for f in (1.0, 1 - 2.0 ** -23, 1 + 2.0 ** -22, 1 - 1e-5, 1 + 1e-5):
        u2 = u.clone()
        u2[:, :2] = (r * f).clamp(0, 1 - 2.0 ** -24).float()
        _check(logits, drafts, u2, draft, 1.0)


def test_given_numbers_at_their_ends():
    logits, drafts, u, draft = _make(5, 12, 3, 301, torch.bfloat16, "sampled", 1.0)
    for value in (0.0, 1 - 2.0 ** -24, 1.0):
        u2 = u.clone()
        u2[:, 3] = value
        want = _check(logits, drafts, u2, draft, 1.0)
        assert bool((want[0].max(1)[0] >= 0).all())
        _check(logits, drafts, torch.full_like(u, value), None, 1.0)
        _check(logits, drafts, torch.full_like(u, value), draft, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mode,T", [("sampled", 0.8), ("lookup", 1.0), ("greedy", 0.0)])
@pytest.mark.parametrize("V", [40, 3007])
def test_odd_rows(dtype, mode, T, V):
    """Masks of -inf and of the type's lowest value, rows of nothing else, NaN, +inf, logits of
    1e30, ties, drafts outside the vocabulary or masked."""
    logits, drafts, u, draft = _make(6, 24, 2, V, dtype, mode, T)
    low = torch.finfo(dtype).min
    x = [logits] + ([draft] if draft is not None else [])
    logits[0, 0, 5:] = -INF
    logits[1, 0, :V - 3] = low
    logits[2, 0] = low
    logits[3, 0] = -INF
    logits[4, 0, 7] = NAN
    logits[5, 1, 7] = INF
    logits[6, 2, V - 1] = NAN
    logits[7, 0] = 1.5
    logits[8] = logits[8].float().mul(1e30).to(dtype)
    drafts[9, 0], drafts[10, 0], drafts[11, 1] = -1, V, 1 << 40
    logits[12, 0, drafts[12, 0]] = -INF
    for t in x:
        t[13, 0, 3] = -INF
        t[14, 0, :V // 2] = -INF
    if draft is not None:
        draft[15, 0, 4] = NAN
        draft[16, 1] = -INF
        draft[17, 0, drafts[17, 0]] = -INF
        draft[18, 0, :] = low
    logits[19, 0] = 0.0
    logits[19, 0, 11] = 0.0
    if V > 30:
        logits[20, :, 20:30] = 30.0
    drafts[20, 0] = 20
    logits[21, 0] = -0.0
    logits[21, 0, 1] = 0.0
    _check(logits, drafts, u, draft, T)


@pytest.mark.parametrize("T", [1e-6, 1e-3, 50.0, 1e6])
def test_temperatures(T):
    logits, drafts, u, draft = _make(7, 20, 3, 1009, torch.float32, "sampled", 1.0)
    _check(logits, drafts, u, draft, T)
    _check(logits, drafts, u, None, T)


def test_strides_streams_and_graphs():
    from naylis_b200 import scoring
    logits, drafts, u, draft = _make(8, 6, 3, 777, torch.bfloat16, "sampled", 1.0)
    want = scoring.verify_drafts(logits, drafts, u, draft_logits=draft)
    wide = torch.randn(6, 5, 900, device=DEV).to(torch.bfloat16)
    wide[:, :4, 50:827] = logits
    got = scoring.verify_drafts(wide[:, :4, 50:827], drafts, u, draft_logits=draft)
    assert torch.equal(got.tokens, want.tokens)
    turned = logits.transpose(0, 1).contiguous().transpose(0, 1)
    cols = logits.transpose(1, 2).contiguous().transpose(1, 2)
    for t in (turned, cols):
        got = scoring.verify_drafts(t, drafts.t().contiguous().t(), u, draft_logits=draft)
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = scoring.verify_drafts(logits, drafts, u, draft_logits=draft)
    side.synchronize()
    assert torch.equal(got.tokens, want.tokens)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = scoring.verify_drafts(logits, drafts, u, draft_logits=draft)
    u.copy_(torch.rand(6, 4, device=DEV))
    g.replay()
    torch.cuda.synchronize()
    now = scoring.verify_drafts(logits, drafts, u, draft_logits=draft)
    assert torch.equal(got.tokens, now.tokens) and torch.equal(got.accepted, now.accepted)


def test_tokens_come_out_as_the_targets():
    """Over a grid of given numbers the first token's frequencies are p: drafts of every kind,
    each with its weight q, 4096 x 64 pairs of numbers each."""
    from naylis_b200 import scoring
    g = torch.Generator().manual_seed(9)
    V, N, M = 6, 1024, 16
    p_logits, q_logits = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = torch.softmax(p_logits.double(), 0), torch.softmax(q_logits.double(), 0)
    u = torch.stack(torch.meshgrid((torch.arange(N) + 0.5) / N, (torch.arange(M) + 0.5) / M, indexing="ij"), -1).view(-1, 2)
    B = N * M
    logits = p_logits.expand(B, 2, V).contiguous().to(DEV)
    draft = q_logits.expand(B, 1, V).contiguous().to(DEV)
    seen = torch.zeros(V, dtype=torch.float64)
    for d in range(V):
        r = scoring.verify_drafts(logits, torch.full((B, 1), d, device=DEV), u.float().to(DEV), draft_logits=draft)
        seen += q[d] * torch.bincount(r.tokens[:, 0].cpu(), minlength=V).double() / B
    # a grid of N numbers counts an interval to 1 / N, one of M to 1 / M of what falls (at most 1)
    assert float((seen - p).abs().max()) < 1 / N + 1 / M


def test_refusals():
    from naylis_b200 import scoring
    x, d, u, q = _make(1, 4, 2, 50, torch.bfloat16, "sampled", 1.0)
    f = scoring.verify_drafts
    f(x, d, u, draft_logits=q)
    for bad in (lambda: f(x.cpu(), d, u), lambda: f(x.half(), d, u), lambda: f(x[0], d, u), lambda: f(x, d[:, :1], u),
                lambda: f(x, d.int(), u), lambda: f(x, d, u.double()), lambda: f(x, d, u[:, :2]), lambda: f(x, d),
                lambda: f(x, d, u, temperature=-1.0), lambda: f(x, d, u, temperature=NAN), lambda: f(x, d, u, temperature=1e7),
                lambda: f(x, d, u, draft_logits=q.float()), lambda: f(x, d, u, draft_logits=q[:, :1]),
                lambda: f(x, d, u, draft_lens=d[:, 0]), lambda: f(x, d.cpu(), u),
                lambda: f(x.repeat(1, 12, 1)[:, :34], d.repeat(1, 17)[:, :33], torch.rand(4, 34, device=DEV))):
        with pytest.raises(RuntimeError):
            bad()
    r = f(x[:0], d[:0], u[:0], draft_logits=q[:0])
    assert r.tokens.shape == (0, 3) and r.accepted.shape == (0,)
