"""Dropout, embedding and sampling through the native host path and through the Python layer: the same outputs and gradients to the bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Watched:
    """The native host path, with a list of whether it took each call."""

    def __init__(self, host):
        self.host, self.taken = host, []

    def __getattr__(self, name):
        def watched(*a):
            out = getattr(self.host, name)(*a)
            self.taken.append(out is not None)
            return out
        return watched


def both(call):
    from pam_b200 import _lib
    watched, results = Watched(_lib.host()), []
    for host in (watched, None):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(_lib, "host", lambda: host)
            results.append(call())
    assert watched.taken and all(watched.taken)
    for a, b in zip(*results, strict=True):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("seed", [5, "tensor", None])
def test_dropout(approx, residual, seed):
    import pam_b200 as pam
    x = torch.randn(33, 65, device="cuda").requires_grad_()
    r = torch.randn(33, 65, device="cuda").requires_grad_() if residual else None
    g = torch.randn(33, 65, device="cuda")
    s = torch.tensor([9], device="cuda") if seed == "tensor" else seed

    def call():
        torch.manual_seed(1)
        y = pam.dropout(x, 0.3, s, r, approx_bwd=approx, offset=1.0625)
        return [y, *torch.autograd.grad(y, [x] + ([r] if residual else []), g)]
    both(call)


@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("p, seed", [(0.0, None), (0.2, 7), (0.2, "tensor"), (0.2, None)])
@pytest.mark.parametrize("positions", [None, "row", "table", "fixed"])
@pytest.mark.parametrize("scale", [None, 3])
def test_embedding(approx, p, seed, positions, scale):
    import pam_b200 as pam
    tokens = torch.randint(0, 50, (4, 9), device="cuda")
    w = torch.randn(50, 36, device="cuda").requires_grad_()
    e = None if positions is None else torch.randn(*((36,) if positions == "row" else (9, 36)), device="cuda").requires_grad_(positions != "fixed")
    g = torch.randn(4, 9, 36, device="cuda")
    s = torch.tensor([9], device="cuda") if seed == "tensor" else seed

    def call():
        torch.manual_seed(1)
        y = pam.embedding(tokens, w, scale, e, 1, p=p, seed=s, approx_bwd=approx)
        return [y, *torch.autograd.grad(y, [w] + ([e] if e is not None and e.requires_grad else []), g)]
    both(call)


def test_sample():
    from pam_b200 import decoding
    x, u = torch.randn(6, 3, 700, device="cuda") * 3, torch.rand(6, 3, device="cuda")
    fill = lambda v: torch.full((6, 3), v, device="cuda")
    banned = torch.rand(700, device="cuda") < 0.2
    for kw in (dict(), dict(temperature=0.5, top_k=9, top_p=0.8, min_p=0.01, banned=banned), dict(temperature=2, top_p=1, min_p=0),
               dict(temperature=fill(0.7), top_k=fill(5), top_p=fill(0.9), min_p=fill(0.05), banned=banned.expand(6, 3, 700).contiguous())):
        both(lambda: decoding.sample(x, u, **kw))


def test_no_product_and_evaluation():
    import pam_b200 as pam
    w = torch.randn(50, 36, device="cuda").requires_grad_()
    tokens = torch.randint(0, 50, (11,), device="cuda")
    both(lambda: [pam.embedding(tokens, w, 2.0, p=0.5, training=False)])
    assert torch.equal(pam.embedding(tokens, w, 2.0, p=0.5, training=False), pam.embedding(tokens, w, 2.0))
    with pytest.raises(ValueError):
        pam.embedding(tokens, w, p=1.5, training=False)
