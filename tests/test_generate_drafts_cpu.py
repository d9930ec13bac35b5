"""CPU tests of what a Session keeps when several tokens are appended and taken back
(naylis_b200/generate.py); the pass is test_generate_cpu's stand-in: a token's id is what
it adds to every router sum."""
import pytest
import torch

from naylis_b200 import attention, generate
from test_generate_cpu import D, LAYERS, V, Fails, _state, session  # noqa: F401


def _sums(s):
    return [t[:, 0].tolist() for t in s.sums]


@pytest.fixture
def undoing(session):  # noqa: F811
    session.undo = 3
    return session


def test_extend_is_steps(undoing):
    s = undoing
    s.add([[1, 2, 3], [4] * 7])
    logits = s.extend(torch.tensor([[5, 6], [7, 8]]))
    assert logits.shape == (2, 2, V) and logits.dtype == torch.bfloat16
    assert [s.cache.length(q) for q in s.seqs] == [5, 9] and _sums(s) == [[17.0, 43.0]] * LAYERS
    logits = s.extend(torch.tensor([[1, 2, 3], [9, 9, 9]]), [3, 1])
    assert _sums(s) == [[23.0, 52.0]] * LAYERS and [s.cache.length(q) for q in s.seqs] == [8, 10]
    assert bool(logits[0].any()) and bool(logits[1, 0].any()) and not logits[1, 1:].any()
    s.extend(torch.tensor([[1], [2]]), [0, 1])
    assert _sums(s) == [[23.0, 54.0]] * LAYERS
    s.step(torch.tensor([1, 1]))
    assert _sums(s) == [[24.0, 55.0]] * LAYERS
    before = _state(s)
    assert s.extend(torch.zeros(2, 0, dtype=torch.int64)).shape == (2, 0, V)
    assert s.extend(torch.ones(2, 2, dtype=torch.int64), [0, 0]).shape == (2, 2, V)
    assert _state(s) == before


def test_retract_takes_back_what_was_appended(undoing):
    s = undoing
    s.add([[1, 2], [3]])
    seen = [_state(s)]
    for a, b in ((4, 5), (6, 7), (8, 9), (1, 2)):
        s.step(torch.tensor([a, b]))
        seen.append(_state(s))
    s.retract([0, 0])
    assert _state(s) == seen[4]
    s.retract([2, 1])
    assert _sums(s) == [[seen[2][3][0][0][0], seen[3][3][0][1][0]]] * LAYERS
    assert [s.cache.length(q) for q in s.seqs] == [4, 4]
    before = _state(s)
    for bad in ([2, 0], [0, 3], [-1, 0], [1], [0, 0, 0]):      # three at most, and two are gone
        with pytest.raises(RuntimeError):
            s.retract(bad)
        assert _state(s) == before
    s.retract([1, 2])
    assert [s.cache.length(q) for q in s.seqs] == [3, 2] and _sums(s) == [[7.0, 8.0]] * LAYERS
    s.extend(torch.tensor([[6, 8, 9], [7, 9, 1]]), [2, 3])
    s.retract([2, 3])
    assert _sums(s) == [[7.0, 8.0]] * LAYERS
    with pytest.raises(RuntimeError):
        s.retract([1, 1])
    # a prompt's tokens stay; one that joined has none yet, one that leaves takes its own along
    s.add([[9]])
    s.step(torch.tensor([1, 1, 1]))
    s.drop([0])
    with pytest.raises(RuntimeError):
        s.retract([0, 2])
    s.retract([1, 1])
    assert _sums(s) == [[8.0, 9.0]] * LAYERS and [s.cache.length(q) for q in s.seqs] == [2, 1]


def test_nothing_to_take_back(session):  # noqa: F811
    s = session
    s.add([[1, 2]])
    s.step(torch.tensor([1]))
    s.retract([0])
    with pytest.raises(RuntimeError):
        s.retract([1])
    with pytest.raises(RuntimeError):
        generate.Session(s.model, 1, undo=-1)


def test_an_extension_that_fails_leaves_the_sequences(undoing):
    s = undoing
    s.add([[1, 2, 3], [4] * 8])
    s.step(torch.tensor([1, 1]))
    before = _state(s)
    tokens = torch.tensor([[7, 9, 1], [9, 2, 3]])
    s.fail = True
    for counts in (None, [1, 3], [0, 2]):
        with pytest.raises(Fails):
            s.extend(tokens, counts)
        assert _state(s) == before
    s.fail = False
    with pytest.raises(RuntimeError, match="pages needed"):
        s.extend(torch.ones(2, 20, dtype=torch.int64))
    for bad, counts in ((torch.tensor([[1], [V]]), None), (torch.tensor([[1], [-1]]), None), (tokens[:1], None),
                        (tokens.float(), None), (tokens[0], None), (tokens, [1]), (tokens, [4, 0]), (tokens, [-1, 1]),
                        (torch.ones(2, attention.MAX_NEW + 1, dtype=torch.int64), None)):
        with pytest.raises(RuntimeError):
            s.extend(bad, counts)
        assert _state(s) == before
    # a token that no count reaches may be anything
    s.extend(torch.tensor([[1, V], [-1, 5]]), [1, 0])
    assert _sums(s) == [[8.0, 33.0]] * LAYERS
    s.retract([2, 1])
    assert _sums(s) == [[6.0, 32.0]] * LAYERS


def test_a_cache_in_4_bits():
    c = attention.PagedKVCache(2, 6, 8, 3, 128, bits=4, device="cpu")
    k, v, scales = c.layer(1)
    assert k.shape == v.shape == (6, 3, 8, 64) and k.dtype == torch.uint8
    assert scales.shape == (6, 3, 8, 2, 4) and scales.dtype == torch.bfloat16
    full = attention.PagedKVCache(2, 6, 8, 3, 128, device="cpu")
    assert len(full.layer(0)) == 2 and full.scales is None
    size = lambda c: sum(t.numel() * t.element_size() for t in c.layer(0))  # noqa: E731
    assert size(c) * 32 == size(full) * 9
    with pytest.raises(RuntimeError):
        attention.PagedKVCache(1, 1, 8, 1, 64, bits=8, device="cpu")


def test_draft_arguments_are_checked():
    for kw in (dict(draft_tokens=0), dict(draft_tokens=33)):
        with pytest.raises(RuntimeError, match="draft_tokens"):
            generate.generate(None, [[1, 2]], 3, draft_model=object(), **kw)
    with pytest.raises(RuntimeError, match="NaylisForCausalLM"):
        generate.generate(None, [[1, 2]], 3, draft_model=torch.nn.Linear(2, 2))
