"""GPU tests of a decoder answering from a 4-bit cache, with several tokens a pass and with a
draft model: append, attention over several new tokens and verification together.

A pass over several tokens and steps of one run the same operators on the same values
with other shapes underneath; logits are held to the bf16 bar of the decoder tests, 2e-2 of
the largest. A cache in 4 bits moves the logits themselves: it is held to the same model
scored with keys and values rounded alike (score(kv_bits=4)), to the same bar."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2e-2


def _model(seed=0, **kw):
    from naylis_b200.decoder import NaylisConfig, NaylisForCausalLM
    torch.manual_seed(seed)
    cfg = NaylisConfig(**{**dict(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=3,
                                 num_attention_heads=4, mem_size=512, mom_block_size=128, mom_top_blocks=2,
                                 mom_router_rank=16), **kw})
    model = NaylisForCausalLM(cfg).cuda().eval()
    with torch.no_grad():
        for m in model.mom_layers():
            m.mom_scale.fill_(0.05)
    return model


def _near(a, b):
    return float((a.float() - b.float()).abs().max() / b.float().abs().max()) < TOL


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("kw", [{}, dict(hidden_size=512)])
def test_extend_matches_steps(bits, kw):
    from naylis_b200 import generate
    model = _model(**kw)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (n,), generator=g).tolist() for n in (1, 17, 300, 128)]
    tail = torch.randint(0, 500, (4, 6), generator=g).cuda()
    one = generate.Session(model, 64, 16, bits)
    many = generate.Session(model, 64, 16, bits, undo=4)
    assert torch.equal(one.add(prompts), many.add(prompts))
    steps = torch.stack([one.step(tail[:, j]) for j in range(6)], 1)
    got = many.extend(tail[:, :4])
    assert _near(got, steps[:, :4])
    # drafts that fall: taken back and replaced
    many.extend((tail[:, :3] + 1) % 500, [1, 3, 0, 2])
    many.retract([1, 3, 0, 2])
    got = many.extend(tail[:, 4:], [2, 1, 2, 0])
    for i, n in enumerate((2, 1, 2, 0)):
        if n:
            assert _near(got[i, :n], steps[i, 4:4 + n])
        assert not got[i, n:].any()
    assert [many.cache.length(q) for q in many.seqs] == [7, 22, 306, 132]
    for a, b in zip(one.sums, many.sums):
        assert _near(b[0], a[0]) and _near(b[2], a[2])


def test_a_cache_in_4_bits_answers_as_it_scores():
    from naylis_b200 import generate
    model = _model(1)
    g = torch.Generator().manual_seed(2)
    seqs = [torch.randint(0, 500, (n,), generator=g).tolist() for n in (40, 9, 333)]
    want = generate.score(model, seqs, kv_bits=4)
    s = generate.Session(model, 64, 16, 4)
    n = 8
    logits = [s.add([p[:-n] for p in seqs])]
    for j in range(n - 1):
        logits.append(s.step(torch.tensor([p[len(p) - n + j] for p in seqs], device="cuda")))
    for i, p in enumerate(seqs):
        rows = torch.stack([x[i] for x in logits]).double()
        lp = torch.log_softmax(rows, -1).gather(1, torch.tensor(p[-n:], device="cuda")[:, None])[:, 0]
        assert float((lp - want[i].logprob[-n:].double()).abs().max()) < 5e-2
    # and near the full cache's, on which 4 bits cost little here
    full = generate.score(model, seqs)
    for a, b in zip(want, full):
        assert float((a.logprob - b.logprob).abs().max()) < 0.5


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("same", [True, False])
def test_greedy_drafts_give_the_models_own_choices(bits, same):
    """Every token is the greatest logit of its own pass, and nearly that of a full one."""
    from naylis_b200 import generate
    model = _model(2)
    helper = model if same else _model(7, num_hidden_layers=1)
    prompts = [[5, 6, 7], [9], list(range(40, 90))]
    out = generate.generate(model, prompts, 13, top_logprobs=2, kv_bits=bits, draft_model=helper, draft_tokens=3)
    again = generate.generate(model, prompts, 13, top_logprobs=2, kv_bits=bits, draft_model=helper, draft_tokens=3)
    for p, a, b in zip(prompts, out, again):
        assert a == b and len(a.tokens) == len(a.logprobs) == len(a.entropies) == len(a.top_ids) == 13
        assert all(t == ids[0] and lp == tl[0] for t, ids, lp, tl in zip(a.tokens, a.top_ids, a.logprobs, a.top_logprobs))
        r = generate.score(model, [p + a.tokens], top_logprobs=1, kv_bits=bits)[0]
        best = r.top_logprob[len(p) - 1:, 0].cpu()
        assert float((torch.tensor(a.logprobs) - best).abs().max()) < 5e-2


def test_drafts_stop_sample_and_refuse():
    from naylis_b200 import generate
    model, helper = _model(3), _model(4, num_hidden_layers=1)
    prompts = [[1, 2, 3], [4, 5], [6]]
    free = generate.generate(model, prompts, 9, draft_model=helper)
    eos = free[0].tokens[2]
    cut = generate.generate(model, prompts, 9, eos_token=eos, draft_model=helper)
    for f, c in zip(free, cut):
        n = f.tokens.index(eos) + 1 if eos in f.tokens else 9
        assert len(c.tokens) == n and c.tokens[:3] == f.tokens[:min(3, n)]

    def sample(seed, **kw):
        return [g.tokens for g in generate.generate(model, prompts, 7, temperature=0.9, draft_model=helper, **kw,
                                                    generator=torch.Generator(device="cuda").manual_seed(seed))]

    assert sample(1) == sample(1) and sample(1) != sample(2)
    assert all(len(t) == 7 for t in sample(3, draft_tokens=8, kv_bits=4))
    for n in (1, 2):
        assert all(len(g.tokens) == n for g in generate.generate(model, prompts, n, draft_model=helper))
    assert generate.generate(model, [], 3, draft_model=helper) == []
    with pytest.raises(RuntimeError, match="tokens"):
        generate.generate(model, prompts, 3, draft_model=_model(5, vocab_size=400))
    with pytest.raises(RuntimeError):
        generate.generate(model, prompts, 3, kv_bits=8)
