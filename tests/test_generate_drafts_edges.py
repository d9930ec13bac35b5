"""CPU tests of generate's and a Session's edges with drafts (naylis_b200/generate.py)."""
import pytest
import torch

from naylis_b200 import generate
from test_generate_cpu import Fails, _state, session  # noqa: F401


def test_the_model_is_checked_before_its_draft_model(monkeypatch):
    """A model of another class is refused in words, whatever drafts for it."""
    draft = object()

    def check(model):
        if model is not draft:
            raise RuntimeError("generate: a NaylisForCausalLM is needed")

    monkeypatch.setattr(generate, "_check_model", check)
    for model in (torch.nn.Linear(2, 2), None):
        with pytest.raises(RuntimeError, match="NaylisForCausalLM"):
            generate.generate(model, [[1, 2]], 3, draft_model=draft)


def test_a_prefill_whose_joins_fail_adds_nothing(session, monkeypatch):  # noqa: F811
    """Whichever allocation of the joined sums fails, the session stays as it was and goes on."""
    s = session
    s.undo = 2
    s.add([[1, 2]])
    s.step(torch.tensor([3]))

    def state():
        return _state(s), [p.tolist() for p in s._past], list(s._known)

    cat, before = torch.cat, state()
    for good in range(20):
        calls = []

        def some(*args, **kw):
            calls.append(0)
            if len(calls) > good:
                raise Fails
            return cat(*args, **kw)

        monkeypatch.setattr(torch, "cat", some)
        try:
            s.add([[4, 5], [6]])
        except Fails:
            monkeypatch.setattr(torch, "cat", cat)
            assert state() == before
            continue
        break
    monkeypatch.setattr(torch, "cat", cat)
    assert good >= 2 * len(s.sums) and [s.cache.length(q) for q in s.seqs] == [3, 2, 1]
    assert s._known == [1, 0, 0] and [len(t) for t in s.sums] == [len(p) for p in s._past] == [3] * len(s.sums)
    s.retract([1, 0, 0])
    assert [t[:, 0].tolist() for t in s.sums] == [[3.0, 9.0, 6.0]] * len(s.sums)


def test_ragged_tokens_come_padded(session):  # noqa: F811
    """Several tokens of each sequence: a tensor with a count for each row; lists of lists are refused."""
    s = session
    s.add([[1, 2], [3]])
    logits = s.extend(torch.tensor([[4, 5, 6], [7, 8, 0]]), counts=[3, 2])
    assert [s.cache.length(q) for q in s.seqs] == [5, 3] and not logits[1, 2].any() and bool(logits[0, 2].any())
    with pytest.raises(RuntimeError, match="tokens must be"):
        s.extend([[4, 5, 6], [7, 8]])
