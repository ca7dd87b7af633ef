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


def _configured(flags, p=0.25):
    import generation_cases as cases
    from pam_b200 import models, steps
    cfgs = models.pam_cfgs()
    torch.manual_seed(0)
    return models.Transformer(steps.TransformerConfig(**cases.CONFIG), linear_cfg=cfgs["linear"], norm_cfg=cfgs["norm"], loss_functional_cfg=cfgs["function"],
                              functional_cfg='{"type": "pam", "dkwargs": {"approx_bwd": %s}}' % flags, dropout=p).cuda()


@pytest.mark.parametrize("flags", ["[true, false]", "[false, true]"])
def test_a_mode_for_each_operand_changes_no_output(flags):
    """Masks and products of the forward pass are those of one mode for both."""
    net, plain = _configured(flags), _configured("true")
    src, out, target = _batch(net)
    results = []
    for model in (net, plain):
        torch.manual_seed(3)
        loss = model.loss(src, out, target)
        loss.backward()
        results.append(loss.detach())
    assert torch.equal(*results)
    assert all(bool(p.grad.isfinite().all()) for p in net.parameters())


@pytest.mark.parametrize("flags, approx", [("[true, false]", True), ("[false, true]", False)])
def test_gradient_has_the_mode_of_the_first_operand(flags, approx):
    import pam_b200 as pam
    from pam_b200 import models
    ops = _configured(flags).decoder.op_dict
    x = (torch.randn(9, 11, generator=torch.Generator().manual_seed(1)) * 3).cuda().requires_grad_()
    g = torch.randn(9, 11, generator=torch.Generator().manual_seed(2)).cuda()
    grads = [torch.autograd.grad(y, x, g)[0] for y in (models._dropped(ops, x, 0.3, 4), pam.dropout(x, 0.3, 4, approx_bwd=approx))]
    assert torch.equal(*grads)


def test_of_shorter_types():
    """What a linear layer under autocast gives is widened, as by the PAM product."""
    import pam_b200 as pam
    from pam_b200 import models
    ops = _configured("true").decoder.op_dict
    x = torch.randn(9, 11).cuda().bfloat16().requires_grad_()
    r = torch.randn(9, 11).cuda()
    y = models._dropped(ops, x, 0.3, 4, r)
    assert y.dtype == torch.float32 and torch.equal(y, pam.dropout(x.detach().float(), 0.3, 4, r))
    (d,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert d.dtype == torch.bfloat16
