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
