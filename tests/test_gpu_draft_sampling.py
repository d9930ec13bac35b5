"""GPU tests of sampling with a draft model (naylis_b200/generate.py): the answers are distributed as
the model's own samples, and a draft model's state follows what stays."""
import pytest
import torch

from test_gpu_drafts import _model

pytestmark = pytest.mark.gpu

V, T, N, NEW = 16, 0.8, 2400, 6


def _small(seed, **kw):
    """A model of 16 tokens with a head of its own (tied to the embedding it would repeat its last token):
    logits about 2 wide, so that no two models are alike and no token is certain."""
    model = _model(seed, vocab_size=V, num_hidden_layers=2, **kw)
    g = torch.Generator().manual_seed(seed + 100)
    model.lm_head.weight = torch.nn.Parameter((torch.randn(V, 256, generator=g) * 0.12).cuda())
    return model


def _counts(model, seed, **kw):
    """Frequencies of the tokens at each place of the answers to one prompt, and of neighbours."""
    from naylis_b200 import generate
    out = generate.generate(model, [[3, 1, 2]] * N, NEW, temperature=T, **kw,
                            generator=torch.Generator(device="cuda").manual_seed(seed))
    tokens = torch.tensor([g.tokens for g in out])
    assert tokens.shape == (N, NEW)
    one = torch.nn.functional.one_hot(tokens, V).double().mean(0)
    pair = torch.nn.functional.one_hot(tokens[:, :-1] * V + tokens[:, 1:], V * V).double().mean(0)
    return one, pair


def _apart(a, b):
    """The greatest difference in units of its own standard deviation (both are means of N)."""
    mean = (a + b) / 2
    return float(((a - b).abs() / (mean * (1 - mean) * 2 / N).sqrt().clamp_min(1.0 / N)).max())


@pytest.mark.parametrize("bits", [16, 4])
def test_answers_are_distributed_as_the_models_own(bits):
    """About 1500 frequencies of 2400 answers: 6 standard deviations of the difference are passed by
    one in 10^6 such tests; the draft model's own answers are far beyond."""
    model, helper = _small(1), _small(2)
    own = _counts(model, 5, kv_bits=bits)
    drafted = _counts(model, 6, kv_bits=bits, draft_model=helper, draft_tokens=3)
    other = _counts(helper, 7, kv_bits=bits)
    assert _apart(own[0], other[0]) > 12
    assert _apart(own[0], drafted[0]) < 6 and _apart(own[1], drafted[1]) < 6


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("other", [False, True])
def test_a_draft_model_follows_what_stays(monkeypatch, bits, other):
    """A model that drafts for itself has nearly every draft kept, in every round (its passes of one and of several
    tokens differ by bf16 roundings), also where the first drafts of each round are made to fall."""
    from naylis_b200 import generate, scoring
    model = _small(1)
    verify, seen = scoring.verify_drafts, []

    def record(logits, drafts, u, *, draft_lens, **kw):
        if other and len(seen) % 2 == 0:      # every second round loses its second draft
            drafts = drafts.clone()
            drafts[:, 1:2] = -1
        got = verify(logits, drafts, u, draft_lens=draft_lens, **kw)
        seen.append((int(got.accepted.sum()), int(draft_lens.sum()), int(draft_lens.clamp_max(1).sum())))
        return got

    monkeypatch.setattr(scoring, "verify_drafts", record)
    prompts = [[3, 1, 2], [5], list(range(16)) * 3] * 40
    out = generate.generate(model, prompts, 24, temperature=T, kv_bits=bits, draft_model=model, draft_tokens=4,
                            generator=torch.Generator(device="cuda").manual_seed(8))
    assert all(len(g.tokens) == 24 for g in out) and len(seen) > 4
    for i, (stay, given, first) in enumerate(seen):
        most = first if other and i % 2 == 0 else given
        assert stay >= 0.9 * most - 4, (i, stay, most, given)
