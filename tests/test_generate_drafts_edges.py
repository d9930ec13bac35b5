"""CPU tests of generate's and a Session's edges with drafts (naylis_b200/generate.py)."""
import pytest
import torch

from naylis_b200 import generate


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
