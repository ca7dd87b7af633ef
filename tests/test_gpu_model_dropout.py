"""The translation model's dropout on the GPU: masks of layers that run again in the backward pass."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_gpu_vocabulary_model import _batch, _dropping

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("whole", [False, True], ids=["encode", "loss"])
def test_checkpointed_layers_draw_the_same_masks(approx, whole):
    net = _dropping(approx=approx)
    src, out, target = _batch(net)

    def step():
        net.zero_grad()
        torch.manual_seed(7)
        total = net.loss(src, out, target) if whole else (net.encode(src) ** 2).sum()
        total.backward()
        return total.detach(), {k: p.grad.clone() for k, p in net.named_parameters() if p.grad is not None}
    want = step()
    for layer in [*net.encoder.layers, *net.decoder.layers]:
        layer.forward = (lambda run: lambda *a, **kw: checkpoint(run, *a, use_reentrant=False, **kw))(layer.forward)
    got = step()
    assert torch.equal(got[0], want[0]) and got[1].keys() == want[1].keys()
    for k, d in got[1].items():
        assert torch.equal(d, want[1][k]), k
