"""GPU tests of generation where something goes wrong: the errors are set or raised on
the host, none of them is a fault of the GPU's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(seed=0):
    from naylis_b200.decoder import NaylisConfig, NaylisForCausalLM
    torch.manual_seed(seed)
    cfg = NaylisConfig(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                       num_attention_heads=4, mem_size=512, mom_block_size=128, mom_top_blocks=2, mom_router_rank=16)
    return NaylisForCausalLM(cfg).cuda().eval()


def test_a_wait_that_gave_up_is_an_error(monkeypatch):
    """The plan's error word, set behind a call: add(), generate() and score() raise,
    and the session goes on as it was."""
    from naylis_b200 import _lib, attention, generate
    model, real = _model(), attention.prompt_attention
    s = generate.Session(model, num_pages=16)
    want = s.add([[1, 2, 3]])

    def gave_up(q, k, v, plan, **kw):
        out = real(q, k, v, plan, **kw)
        plan.list_for(q.shape[1], k.shape[1])[:4].view(torch.int32).fill_(2)
        return out

    with monkeypatch.context() as m:
        m.setattr(attention, "prompt_attention", gave_up)
        for call in (lambda: s.add([[4, 5]]), lambda: generate.generate(model, [[1, 2]], 2),
                     lambda: generate.score(model, [[1, 2, 3]])):
            with pytest.raises(_lib.MomError, match="gave up"):
                call()
    assert len(s.seqs) == 1 and s.cache.free_pages == 15
    assert torch.equal(s.add([[1, 2, 3]]), want)


def test_a_failed_step_can_be_taken_again(monkeypatch):
    """The pass fails behind its first layer's attention; the step after it gives what it
    would have given."""
    from naylis_b200 import attention, generate
    model, real = _model(1), attention.decode_attention
    prompts, tokens = [list(range(1, 17)), [7, 8, 9]], torch.tensor([3, 4], device="cuda")
    s, other = generate.Session(model, num_pages=16), generate.Session(model, num_pages=16)
    s.add(prompts)
    other.add(prompts)
    calls = []

    def fails(*a, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise MemoryError
        return real(*a, **kw)

    with monkeypatch.context() as m:
        m.setattr(attention, "decode_attention", fails)
        with pytest.raises(MemoryError):
            s.step(tokens)
    assert [s.cache.length(q) for q in s.seqs] == [16, 3]
    for _ in range(2):
        assert torch.equal(s.step(tokens), other.step(tokens))
