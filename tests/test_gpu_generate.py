"""GPU tests of generation (naylis_b200/generate.py) against the training forward
over the whole sequence: each step's logits, the chosen tokens and their scores.

Both sides run the trunk in bf16 with different products underneath (one pass over
all positions and torch's attention, against packed prefill and cached steps), so
logits are held to the bf16 bar of the decoder tests, 2e-2 of the largest. Scores
are held to the same logits' log-softmax in 64 bits."""
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


def _full(model, ids):
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        return model(torch.tensor([ids], device="cuda"))[0].float()


@pytest.mark.parametrize("kw", [{}, dict(hidden_size=512, num_attention_heads=4), dict(num_hidden_layers=1)])
def test_prefill_and_steps_match_the_full_pass(kw):
    from naylis_b200 import generate
    model = _model(**kw)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (n,), generator=g).tolist() for n in (1, 17, 300, 128)]
    tail = torch.randint(0, 500, (6, 4), generator=g)
    s = generate.Session(model, num_pages=64, page_size=16)
    logits = s.add(prompts)
    for step in range(7):
        for i, p in enumerate(prompts):
            want = _full(model, p + tail[:step, i].tolist())[-1]
            err = float((logits[i].float() - want).abs().max() / want.abs().max())
            assert err < TOL, (step, i, err)
        if step < 6:
            logits = s.step(tail[step].cuda())
    assert [s.cache.length(q) for q in s.seqs] == [7, 23, 306, 134]
    # a sequence that joins later, and one that leaves
    s.drop([1])
    more = s.add([prompts[1] + tail[:6, 1].tolist()])
    want = _full(model, prompts[1] + tail[:6, 1].tolist())[-1]
    assert float((more[0].float() - want).abs().max() / want.abs().max()) < TOL
    nxt = s.step(torch.tensor([3, 4, 5, 6], device="cuda"))
    for i, ids in enumerate([prompts[0] + tail[:6, 0].tolist() + [3], prompts[2] + tail[:6, 2].tolist() + [4],
                             prompts[3] + tail[:6, 3].tolist() + [5], prompts[1] + tail[:6, 1].tolist() + [6]]):
        want = _full(model, ids)[-1]
        assert float((nxt[i].float() - want).abs().max() / want.abs().max()) < TOL


def test_generate_scores_its_tokens():
    from naylis_b200 import generate
    model = _model(2)
    prompts = [[5, 6, 7], [9], list(range(40, 90))]
    out = generate.generate(model, prompts, 12, top_logprobs=4)
    again = generate.generate(model, prompts, 12, top_logprobs=4)
    for p, g, g2 in zip(prompts, out, again):
        assert g == g2 and len(g.tokens) == len(g.logprobs) == len(g.top_ids) == 12
        assert all(t == ids[0] and lp == tl[0] for t, ids, lp, tl in zip(g.tokens, g.top_ids, g.logprobs, g.top_logprobs))
        # the scores of the finished text from one packed pass: the same distributions through other products
        r = generate.score(model, [p + g.tokens], top_logprobs=1)[0]
        want = r.logprob[len(p) - 1:].cpu()
        assert float((torch.tensor(g.logprobs) - want).abs().max()) < 5e-2
        full = _full(model, p + g.tokens)
        lp = torch.log_softmax(full.double(), -1)[:-1].gather(1, torch.tensor(p + g.tokens, device="cuda")[1:, None])[:, 0]
        assert float((r.logprob.double() - lp).abs().max()) < 5e-2


def test_generate_stops_samples_and_refuses():
    from naylis_b200 import generate
    model = _model(3)
    prompts = [[1, 2, 3], [4, 5], [6]]
    free = generate.generate(model, prompts, 8)
    eos = free[0].tokens[2]
    cut = generate.generate(model, prompts, 8, eos_token=eos)
    for f, c in zip(free, cut):
        n = f.tokens.index(eos) + 1 if eos in f.tokens else 8
        assert len(c.tokens) == n and c.tokens[:3] == f.tokens[:min(3, n)]
    def sample(seed):
        return generate.generate(model, prompts, 5, temperature=0.8,
                                 generator=torch.Generator(device="cuda").manual_seed(seed))
    assert [g.tokens for g in sample(1)] == [g.tokens for g in sample(1)]
    assert [g.tokens for g in sample(1)] != [g.tokens for g in sample(2)]
    assert generate.generate(model, [], 3) == [] and generate.generate(model, prompts, 0)[0].tokens == []
    for bad in ([[]], [[500]], [[-1]]):
        with pytest.raises(RuntimeError):
            generate.generate(model, bad, 2)
    with pytest.raises(RuntimeError):
        generate.generate(model, prompts, 2, temperature=-1.0)
    with pytest.raises(RuntimeError):
        generate.generate(model, [[1] * 40], 2, num_pages=2)
    with pytest.raises(RuntimeError):
        generate.generate(_model(4, scan_mode="fp64"), prompts, 2)
    s = generate.Session(model, num_pages=2, page_size=8)
    s.add([[1] * 16])
    with pytest.raises(RuntimeError):
        s.step(torch.tensor([1], device="cuda"))
    assert s.cache.length(s.seqs[0]) == 16 and s.cache.free_pages == 0
    s.drop([0])
    assert s.cache.free_pages == 2
