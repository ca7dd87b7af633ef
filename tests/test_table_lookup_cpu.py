"""When the translation model looks tokens up by the fused operator, on the CPU with a stand-in for it."""
import pytest
import torch
from torch import nn

import generation_cases as cases


@pytest.fixture
def stack(monkeypatch):
    """An encoder whose fused lookups are counted in `stack.fused`."""
    from pam_b200 import models, pam_ops
    net = cases.model({}, "cpu")
    net.encoder.fused = []
    monkeypatch.setattr(models, "_scaling", lambda ops, t: {})

    def embedding(tokens, weight, scale, positions, padding_idx, *, p=0.0, seed=None):
        net.encoder.fused.append(p)
        return nn.functional.embedding(tokens, weight, padding_idx) * scale + positions
    monkeypatch.setattr(pam_ops, "embedding", embedding)
    return net.encoder


TOKENS = torch.tensor([[4, 9, 7], [1, 5, 9]])
KINDS = {
    "max_norm": lambda t: setattr(t, "max_norm", 0.5),
    "sparse": lambda t: setattr(t, "sparse", True),
    "scale_grad_by_freq": lambda t: setattr(t, "scale_grad_by_freq", True),
    "own forward": lambda t: setattr(t, "forward", lambda tokens: nn.functional.embedding(tokens, t.weight) + 1),
}


def test_plain_tables(stack):
    stack.embed(TOKENS)
    assert not stack.fused                                    # (a training step without dropout)
    with torch.no_grad():
        stack.embed(TOKENS)
    stack.dropout = 0.2
    stack.embed(TOKENS)
    assert stack.fused == [0.0, 0.2]


@pytest.mark.parametrize("kind", KINDS)
def test_tables_of_another_kind_look_up_themselves(stack, kind):
    KINDS[kind](stack.embed_tokens)
    want = stack.embed(TOKENS).detach()
    with torch.no_grad():
        assert torch.equal(stack.embed(TOKENS), want)
    stack.dropout = 0.2
    stack.embed(TOKENS)
    assert not stack.fused


HOOKS = ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"]


@pytest.mark.parametrize("name", HOOKS)
@pytest.mark.parametrize("everywhere", [False, True], ids=["table", "all modules"])
def test_hooks_are_called(stack, name, everywhere):
    calls = []
    hook = lambda module, *a: calls.append(module)
    handle = getattr(nn.modules.module, name.replace("register_", "register_module_")) if everywhere else getattr(stack.embed_tokens, name)
    handle = handle(hook)
    try:
        stack.dropout = 0.2
        stack.embed(TOKENS).sum().backward()
    finally:
        handle.remove()
    assert calls == [stack.embed_tokens] and not stack.fused
