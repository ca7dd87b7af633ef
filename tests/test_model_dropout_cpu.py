"""The translation model's dropout on the CPU, with a stand-in whose mask follows its seed alone, as on a GPU."""
import types

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import generation_cases as cases


@pytest.fixture
def net(monkeypatch):
    """A model in training whose steps draw their seeds as they do for a GPU."""
    from pam_b200 import models, steps

    def dropped(ops, x, p, seed, residual=None):
        kept = torch.rand(x.shape, generator=torch.Generator().manual_seed(int(seed) % 2 ** 63)) >= p
        x = x * kept / (1 - p)
        return x if residual is None else residual + x
    draw, seeds = torch.randint, models.Transformer._seeds
    monkeypatch.setattr(models, "_dropped", dropped)
    monkeypatch.setattr(torch, "randint", lambda low, high, size, device=None: draw(low, high, size))
    monkeypatch.setattr(models.Transformer, "_seeds", lambda self, device: seeds(self, types.SimpleNamespace(type="cuda")))
    torch.manual_seed(0)
    return models.Transformer(steps.TransformerConfig(**cases.CONFIG), dropout=0.3)


def _gradients(net, call):
    net.zero_grad()
    torch.manual_seed(3)
    out = call()
    (out * out).sum().backward()
    return out.detach(), {name: p.grad.clone() for name, p in net.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("whole", [False, True], ids=["encode", "forward"])
def test_checkpointed_layers_draw_the_same_masks(net, whole):
    src, out = torch.full((2, 5), 7), torch.full((2, 4), 9)
    call = (lambda: net(src, out)) if whole else (lambda: net.encode(src))
    want = _gradients(net, call)
    for layer in [*net.encoder.layers, *net.decoder.layers]:
        layer.forward = (lambda run: lambda *a, **kw: checkpoint(run, *a, use_reentrant=False, **kw))(layer.forward)
    got = _gradients(net, call)
    assert torch.equal(got[0], want[0]) and got[1].keys() == want[1].keys()
    for name, d in got[1].items():
        assert torch.equal(d, want[1][name]), name


def test_each_mask_has_a_seed_of_its_own(net, monkeypatch):
    from pam_b200 import models
    seeds, dropped = [], models._dropped

    def counted(ops, x, p, seed, residual=None):
        seeds.append(int(seed))
        return dropped(ops, x, p, seed, residual)
    monkeypatch.setattr(models, "_dropped", counted)
    net(torch.full((2, 5), 7), torch.full((2, 4), 9))
    # the embeddings, two sublayers of an encoder layer and three of a decoder layer
    assert len(seeds) == len(set(seeds)) == 2 + 2 * 2 + 3 * 2


@pytest.mark.parametrize("flags, first", [((True, False), True), ((False, True), False), (True, True), ((False, False), False)], ids=str)
def test_a_pam_dictionary_has_a_pam_dropout(monkeypatch, flags, first):
    """Whatever its gradient mode and the tensors' type: never the ordinary product."""
    from pam_b200 import factories, models, pam_ops
    name = lambda v: str(v).lower()
    mode = name(flags) if isinstance(flags, bool) else "[" + ", ".join(map(name, flags)) + "]"
    ops = factories.get_function_dict('{"type": "pam", "dkwargs": {"approx_bwd": %s}}' % mode)
    assert models._pam_binding(ops, ("mul",)) is not None
    calls = []
    monkeypatch.setattr(pam_ops, "dropout", lambda x, p, seed, residual, **kw: calls.append((x, p, seed, residual, kw)) or x)
    monkeypatch.setattr(models.F, "dropout", lambda *a, **kw: pytest.fail("an ordinary dropout"))
    x, r = torch.randn(3, 4), torch.randn(3, 4)
    models._dropped(ops, x, 0.3, 5, r)
    models._dropped(ops, x.bfloat16(), 0.3, None)
    for (got, p, seed, residual, kw), want in zip(calls, ((x, 5, r), (x.bfloat16().float(), None, None))):
        assert got.dtype == torch.float32 and torch.equal(got, want[0]) and (p, seed) == (0.3, want[1]) and residual is want[2]
        assert _flag(kw["approx_bwd"]) is first and kw.get("offset") in (None, 1.0)


def _flag(approx_bwd):
    return approx_bwd if isinstance(approx_bwd, bool) else (set(approx_bwd).pop() if len(set(approx_bwd)) == 1 else None)


def test_other_dictionaries_have_the_ordinary_one():
    from pam_b200 import models
    x, r = torch.randn(3, 4), torch.randn(3, 4)
    torch.manual_seed(1)
    got = models._dropped(dict(mul=torch.mul), x, 0.3, None, r)
    torch.manual_seed(1)
    assert torch.equal(got, r + torch.nn.functional.dropout(x, 0.3))
