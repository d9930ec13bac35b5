"""CPU tests of a Session's book-keeping (naylis_b200/generate.py): the trunk's pass is a
stand-in, its failures are raised on the host."""
import types

import pytest
import torch

from naylis_b200 import attention, generate

D, V, LAYERS = 4, 11, 2


class Fails(Exception):
    pass


@pytest.fixture
def session(monkeypatch):
    """A Session on the CPU whose pass files nothing, adds each token's id to every layer's
    router sum and returns hidden states of 1. `session.fail` makes it raise behind the
    first layer."""
    monkeypatch.setattr(generate, "_check_model", lambda model: None)
    monkeypatch.setattr(generate.trunk, "bank_kv", lambda *a: None)
    monkeypatch.setattr(generate.trunk, "linear_f32grad", lambda x, w: (x @ w.t()).bfloat16())
    mom = types.SimpleNamespace(k_proj=types.SimpleNamespace(weight=None), v_proj=types.SimpleNamespace(weight=None),
                                mem_slots=0, router_down=types.SimpleNamespace(weight=None),
                                router_up=types.SimpleNamespace(weight=None), top_blocks=1)
    layers = [types.SimpleNamespace(mom=mom) for _ in range(LAYERS)]
    model = types.SimpleNamespace(
        config=types.SimpleNamespace(num_hidden_layers=LAYERS, num_attention_heads=2, head_dim=64, vocab_size=V),
        model=types.SimpleNamespace(embed_tokens=types.SimpleNamespace(weight=torch.ones(V, D)), layers=layers,
                                    M_blocks=None),
        lm_head=types.SimpleNamespace(weight=torch.ones(V, D)))

    class Ops:
        def __init__(self, *a):
            pass

        def zero_carry(self, x, mode):
            return None

        def route(self, x, *a):
            return None, torch.zeros(1, x.shape[1], 1), torch.ones(1, x.shape[1], 1), x.sum(1)

    monkeypatch.setattr(generate, "CudaShardOps", Ops)
    monkeypatch.setattr(generate.mk, "mom_route_log_gates",
                        lambda mean, *a: (None, torch.zeros(len(mean), 1, 1), None, torch.zeros(len(mean), 1, 1)))
    s = generate.Session(model, num_pages=4, page_size=8)
    s.fail = False

    def run(ids, positions, slots, longest, attend, route, want_k):
        assert len(ids) == len(positions) == len(slots)
        y32 = ids.float()[:, None].expand(-1, D)
        for i in range(LAYERS):
            route(i, mom, y32)
            if s.fail:
                raise Fails
        return torch.ones(len(ids), D)

    monkeypatch.setattr(s, "_pass", run)
    return s


def _state(s):
    return (list(s.seqs), [s.cache.length(q) for q in s.seqs], s.cache.free_pages,
            None if s.sums is None else [t.tolist() for t in s.sums])


def test_a_prefill_that_fails_adds_nothing(session):
    s = session
    for prompts, error in (([[1, 2, 3]], Fails), ([[1] * 9, [2] * 33], RuntimeError)):
        s.fail = error is Fails
        before = _state(s)
        with pytest.raises(error):
            s.add(prompts)
        assert _state(s) == before
    s.fail = False
    s.add([[1, 2, 3], [4] * 9])
    assert _state(s) == (s.seqs, [3, 9], 1, [[[6.0] * D, [36.0] * D]] * LAYERS)
    s.fail = True
    before = _state(s)
    with pytest.raises(Fails):
        s.add([[5]])
    assert _state(s) == before


def test_a_step_that_fails_leaves_the_sequences(session):
    """Lengths, pages and the router's sums stay, also where the token would have begun a
    page; the same step then goes through."""
    s = session
    s.add([[1, 2, 3], [4] * 8])
    tokens = torch.tensor([7, 9])
    before = _state(s)
    s.fail = True
    for _ in range(3):
        with pytest.raises(Fails):
            s.step(tokens)
        assert _state(s) == before
    s.fail = False
    logits = s.step(tokens)
    assert logits.shape == (2, V)
    assert _state(s) == (s.seqs, [4, 9], 1, [[[13.0] * D, [41.0] * D]] * LAYERS)


def test_retract():
    c = attention.PagedKVCache(1, 4, 8, 1, 64, device="cpu")
    a, b = c.add(), c.add()
    c.extend([a, b], [8, 3])
    first = c.extend([a, b], [9, 1])
    c.retract([a, b], [9, 1])
    assert (c.length(a), c.length(b), c.free_pages) == (8, 3, 2)
    assert [t.tolist() for t in c.extend([a, b], [9, 1])] == [t.tolist() for t in first]
    for seqs, counts in (([a, b], [1, 5]), ([a], [-1]), ([a, a], [1, 1]), ([a], [])):
        with pytest.raises(RuntimeError):
            c.retract(seqs, counts)
    assert (c.length(a), c.length(b), c.free_pages) == (17, 4, 0)
    c.retract([a, b], [17, 4])
    assert c.free_pages == 4


def test_drop_takes_rows_that_there_are(session):
    s = session
    assert s.drop([]).tolist() == []
    s.add([[1], [2] * 9, [3]])
    before = _state(s)
    for rows in ([-1], [3], [0, 5], [1, -3]):
        with pytest.raises(RuntimeError):
            s.drop(rows)
        assert _state(s) == before
    with pytest.raises(TypeError):
        s.drop([1.5])
    assert _state(s) == before
    last = s.seqs[2]
    assert s.drop([0, 1, 1]).tolist() == [2]
    assert _state(s) == ([last], [1], 3, [[[3.0] * D]] * LAYERS)


class _Plan:
    """A PromptPlan that a wait of the attention gave up on, `times` times."""
    times = 0

    def __init__(self, lens, device):
        pass

    def check(self):
        if _Plan.times > 0:
            _Plan.times -= 1
            raise attention._lib.MomError(6, "mom_prompt_plan_check", "a bounded device-side wait gave up")


def test_a_wait_that_gave_up_is_an_error(session, monkeypatch):
    monkeypatch.setattr(generate.attention, "PromptPlan", _Plan)
    s, _Plan.times = session, 1
    before = _state(s)
    with pytest.raises(attention._lib.MomError):
        s.add([[1, 2]])
    assert _state(s) == before and _Plan.times == 0
    assert s.add([[1, 2]]).shape == (1, V)

    monkeypatch.setattr(generate, "Session", lambda *a: session)
    monkeypatch.setattr(generate.scoring, "token_logprobs", lambda x, t, **kw: (t.float(), t.float(), None, None))
    _Plan.times = 1
    with pytest.raises(attention._lib.MomError):
        generate.score(session.model, [[1, 2, 3]])
    assert generate.score(session.model, [[1, 2, 3], [4, 5]])[1].logprob.tolist() == [5.0]


def test_step_refuses_what_the_embedding_would_fault_on(session):
    s = session
    s.add([[1, 2], [3]])
    before = _state(s)
    for tokens in (torch.tensor([1, V]), torch.tensor([-1, 1]), torch.tensor([1 << 40, 1]), torch.tensor([1]),
                   torch.tensor([1, 2, 3]), torch.tensor([[1, 2]]), torch.tensor([1.0, 2.0]),
                   torch.tensor([True, False]), [1, 2]):
        with pytest.raises(RuntimeError):
            s.step(tokens)
        assert _state(s) == before
    s.step(torch.tensor([0, V - 1]))
    s.step(torch.tensor([0, V - 1], dtype=torch.int32))
    assert [s.cache.length(q) for q in s.seqs] == [4, 3]


def test_step_without_sequences(session):
    """Before the first and behind the last: no rows, no pass."""
    s, none = session, torch.zeros(0, dtype=torch.int64)
    s.fail = True
    assert s.step(none).shape == (0, V) and s.step(none).dtype == torch.bfloat16
    s.fail = False
    s.add([[1, 2]])
    s.drop([0])
    s.fail = True
    assert s.step(none).shape == (0, V) and s.cache.free_pages == 4


def test_models_that_cannot_answer_are_refused():
    from naylis_b200.decoder import NaylisConfig, NaylisForCausalLM
    cfg = NaylisConfig(vocab_size=16, hidden_size=128, intermediate_size=128, num_hidden_layers=1,
                       num_attention_heads=2, mem_size=128, mom_block_size=128, mom_top_blocks=1, mom_router_rank=8)
    for model in (None, torch.nn.Linear(2, 2), NaylisForCausalLM(cfg)):      # the last is on the CPU
        for call in (lambda: generate.Session(model, 1), lambda: generate.generate(model, [[1]], 1),
                     lambda: generate.score(model, [[1, 2]])):
            with pytest.raises(RuntimeError, match="NaylisForCausalLM"):
                call()


def test_page_sizes_are_checked_before_they_are_used():
    for size in (0, -8, 12, 512):
        with pytest.raises(RuntimeError, match="page_size"):
            generate.generate(None, [[1, 2]], 3, page_size=size)
