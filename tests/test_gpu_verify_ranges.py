"""GPU tests of scoring.verify_drafts where its parts meet: drafts that fall although both rows are
one distribution, vocabularies whose terms are not kept, sums that 32 bits do not hold."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_verify import DEV, INF, NAN, _check, _make  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ nothing left of the target
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(9, 1000), (40, 257), (9, 40000), (300, 4999)])
@pytest.mark.parametrize("shift", [0.0, 8.0])
def test_a_draft_falls_between_equal_rows(dtype, B, V, shift):
    """The draft's distribution is the target's, and its draft falls all the same (outside the vocabulary, masked
    in both rows, or a given number of 1): nothing is left, and the token is the target's own."""
    K = 2
    g = torch.Generator().manual_seed(V)
    # quarters up to 16: a shift of 8 is exact in bf16
    logits = (torch.randn(B, K + 1, V, generator=g) * 6).round().clamp(-28, 28) / 4
    logits = logits.to(dtype).to(DEV)
    drafts = torch.randint(0, V, (B, K), generator=g).to(DEV)
    u = torch.rand(B, K + 1, generator=g).to(DEV)
    u[0::4, 0] = 1.0
    drafts[1::4, 0] = -1
    drafts[2::4, 0] = V
    for b in range(3, B, 4):
        logits[b, 0, drafts[b, 0]] = -INF
    u[4::5, 1] = 1.0
    draft = logits[:, :K] + shift
    want = _check(logits, drafts, u, draft, 1.0)
    assert not want[1][:4].any() and len(set(want[0][:, 0].tolist())) > 4
    if shift == 0.0:
        _check(logits, drafts, u, draft, 0.7)

# ------------------------------------------------------------------ sums that 32 bits do not hold
def test_sums_of_very_large_vocabularies():
    """Rows of two values: a lane's 32-bit sum of 32768 equal terms is off by up to 2^-11 of it, as every
    addition rounds the same way. Drafts are tested at given numbers 2^-11.. 2^-13 beside p."""
    from naylis_b200 import scoring
    V, K, B, high = 1 << 21, 7, 256, 4096
    gaps = torch.tensor([1.0, 1.25, 1.5, 2.0, 2.25, 3.0, 3.5, 0.75])
    x = torch.zeros(K + 1, V) - gaps[:, None]
    x[:, :high] = 0.0
    logits = x.to(torch.bfloat16).to(DEV).expand(B, K + 1, V)
    p = 1.0 / (high + (V - high) * torch.exp(-gaps.double()))
    drafts = torch.arange(B * K).view(B, K) % high      # of the likely ones
    u = torch.zeros(B, K + 1)
    u[:, K] = 0.5
    want = torch.empty(B, dtype=torch.int64)
    for b in range(B):
        j, f = b % K, 2.0 ** (-11 - (b // K) % 9 / 4) * (1 if b // (9 * K) % 2 else -1)
        u[b, j] = float(p[j] * (1 + f))
        u[b, j + 1:K] = 1.0
        want[b] = j + int(float(u[b, j]) < float(p[j]))
    got = scoring.verify_drafts(logits, drafts.to(DEV), u.to(DEV))
    assert torch.equal(got.accepted.cpu(), want), (got.accepted.cpu() != want).nonzero()[:, 0].tolist()

# ------------------------------------------------------------------ terms that are not kept
NOT_KEPT = [("sampled", 9, 2, 40000), ("sampled", 600, 2, 5001), ("lookup", 9, 2, 70001), ("lookup", 600, 1, 9001)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mode,B,K,V", NOT_KEPT)
def test_vocabularies_that_are_not_kept(dtype, mode, B, K, V):
    """A CTA's stretch of the rows is more than its shared memory holds: terms are computed where they are needed."""
    logits, drafts, u, draft = _make(B + V, B, K, V, dtype, mode, 0.8)
    logits[0, 0, V // 3:] = -INF
    logits[1, 0, :V - 5] = torch.finfo(dtype).min
    logits[2, 0, 11] = NAN
    logits[3, 0] = -INF
    logits[4, 0] = 0.25
    drafts[5, 0], drafts[6, 0] = -1, V
    logits[7, 0, drafts[7, 0]] = -INF
    if draft is not None:
        draft[8, 0] = logits[8, 0]
        draft[3, 1], draft[4, 0] = -INF, 0.25
    want = _check(logits, drafts, u, draft, 0.8)
    if B > 9:      # the inputs reach every end
        assert len(set(want[1].tolist())) > 1
    _check(logits, drafts, u, draft, 0.8, [(3 * i) % (K + 1) for i in range(B)])
    for value in (0.0, 1 - 2.0 ** -24):
        u2 = u.clone()
        u2[:, K] = value
        _check(logits, drafts, u2, draft, 0.8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("own", [False, True])
def test_borders_that_are_not_kept(dtype, own):
    """Given numbers at p / q, where 32-bit sums leave the draft open."""
    B, K, V = (9, 2, 40009) if own else (9, 2, 70001)
    logits, drafts, u, draft = _make(5, B, K, V, dtype, "sampled" if own else "lookup", 1.0, noise=2.0)
    r = torch.softmax(logits[:, :K].double(), -1).gather(2, drafts[..., None])[..., 0]
    if own:
        r = r / torch.softmax(draft.double(), -1).gather(2, drafts[..., None])[..., 0]
    for f in (1.0, 1 - 2.0 ** -23, 1 + 2.0 ** -22, 1 - 1e-5, 1 + 1e-5):
        u2 = u.clone()
        u2[:, :K] = (r * f).clamp(0, 1 - 2.0 ** -24).float()
        _check(logits, drafts, u2, draft, 1.0)


# ------------------------------------------------------------------ clusters of either size
@pytest.mark.parametrize("mode,T", [("sampled", 1.0), ("lookup", 1.0), ("greedy", 0.0)])
@pytest.mark.parametrize("V", [5003, 40000])
def test_a_sequence_alone_and_in_a_batch(mode, T, V):
    """Clusters of 16 CTAs alone, of 8 and fewer among others: the same tokens."""
    from naylis_b200 import scoring
    logits, drafts, u, draft = _make(V, 70, 3, V, torch.bfloat16, mode, T)

    def run(rows):
        return scoring.verify_drafts(logits[rows], drafts[rows], None if u is None else u[rows], temperature=T,
                                     draft_logits=None if draft is None else draft[rows])

    every = run(slice(0, 70))
    for n in (1, 8, 9, 30):
        got = run(slice(0, n))
        assert torch.equal(got.tokens, every.tokens[:n]) and torch.equal(got.accepted, every.accepted[:n])


def test_a_first_call_that_is_captured():
    """A process whose first calls are captured: what they ask of the device once does not disturb it."""
    code = """
import torch
from naylis_b200 import scoring
for dtype in (torch.bfloat16, torch.float32):
    x, q = torch.randn(3, 3, 500, device="cuda").to(dtype), torch.randn(3, 2, 500, device="cuda").to(dtype)
    d, u = torch.randint(0, 500, (3, 2), device="cuda"), torch.rand(3, 3, device="cuda")
    torch.cuda.synchronize()
    for args, kw in (((x, d, u), dict(draft_logits=q)), ((x, d, u), {}), ((x, d), dict(temperature=0.0))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = scoring.verify_drafts(*args, **kw)
        g.replay()
        torch.cuda.synchronize()
        now = scoring.verify_drafts(*args, **kw)
        assert torch.equal(got.tokens, now.tokens) and torch.equal(got.accepted, now.accepted)
print("fine")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-2000:]
