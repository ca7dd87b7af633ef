"""Dropout on the GPU against its definition: the kept elements and the products to the bit, with a residual to one rounding."""
import pytest
import torch

import vocabulary_cases as define
from conftest import assert_bits_equal

pytestmark = pytest.mark.gpu
U = define.U


@pytest.fixture(scope="module")
def pam():
    import pam_b200
    return pam_b200


def data(n, seed=0, special=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g)
    if special:
        some = torch.tensor([0.0, -0.0, 1e-37, -2e-37, 1e-45, 3e36, -9e36, 1e38, 0.7])
        x[torch.randint(0, n, (n // 4 + 1,), generator=g)] = some[torch.randint(0, len(some), (n // 4 + 1,), generator=g)]
    return x


@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n, p, seed", [(1, 0.5, 0), (3, 0.1, 1), (4, 0.3, -1), (5, 0.9, 2 ** 63 - 1), (1023, 0.001, 7), (2048, 0.5, -2 ** 63), (4097, 0.999, 12345678901),
                                        (100003, 0.3, 42)])
def test_against_definition(pam, n, p, seed, residual, approx):
    x, g, r = data(n, 1, special=True), data(n, 2, special=True), data(n, 3)
    xd = x.cuda().requires_grad_()
    rd = r.cuda().requires_grad_() if residual else None
    out = pam.dropout(xd, p, seed, rd, approx_bwd=approx)
    want, mask = define.dropped(x, p, seed)
    if residual:
        total = want + r.double()
        near = (out.double().cpu() - total).abs() <= U * total.abs()
        assert bool((near | (total.isnan() & out.isnan().cpu())).all())
    else:
        assert_bits_equal(out, want.float())
    grads = torch.autograd.grad(out, [xd] + ([rd] if residual else []), g.cuda())
    if approx:
        assert_bits_equal(grads[0], define.dropped_grad(g, x, p, seed, True).float())
    else:
        # (slopes of zeros, of denormals and of what the range rule cuts off are patterns that the scalar functions define: pam_bwd)
        slopes = pam.cuda_bindings.cuda_kernels.pam_bwd(x.cuda(), torch.full((n,), define.scale_of(p)).cuda(), g.cuda(), 1.0)
        assert_bits_equal(grads[0], torch.where(mask, slopes.cpu(), 0.0))
        plain = (x.abs() > 1e-30) & (x.abs() < 1e30) & (g.abs() < 1e36) & (g.abs() > 1e-36)
        assert_bits_equal(grads[0].cpu()[plain], define.dropped_grad(g, x, p, seed, False).float()[plain])
    if residual:
        assert_bits_equal(grads[1], g)


def test_gradient_against_differences(pam):
    # (away from the kinks of the PAM product: a step of 2^-12 of the value within one piece)
    x = (1.0 + torch.arange(64) / 256.0 + 2 ** -10).cuda().requires_grad_()
    out = pam.dropout(x, 0.25, 3)
    (d,) = torch.autograd.grad(out.sum(), x)
    h = 2.0 ** -12
    with torch.no_grad():
        steps = (pam.dropout(x + h, 0.25, 3) - pam.dropout(x, 0.25, 3)) / h
    assert torch.equal(d, steps)


@pytest.mark.parametrize("make", [lambda x: x[1:1 + 4000], lambda x: x[:4096].view(64, 64).t(), lambda x: x[:4000:2], lambda x: x[:1].expand(33, 5)])
def test_layouts(pam, make):
    """A mask goes by an element's place in the tensor, whatever its strides and addresses."""
    x = make(data(8192, 4))
    out = pam.dropout(make(data(8192, 4).cuda()), 0.4, 99)
    want, _ = define.dropped(x.contiguous(), 0.4, 99)
    assert_bits_equal(out, want.float())
    r = torch.randn(x.shape).cuda()
    shifted = torch.randn(x.numel() + 1).cuda()[1:].view(x.shape)
    assert torch.equal(pam.dropout(shifted, 0.4, 99, r), pam.dropout(shifted.clone(), 0.4, 99) + r)


def test_seeds(pam):
    x = torch.ones(1000).cuda()
    assert torch.equal(pam.dropout(x, 0.5, 17), pam.dropout(x, 0.5, torch.tensor([17]).cuda()))
    assert torch.equal(pam.dropout(x, 0.5, 17), pam.dropout(x, 0.5, torch.tensor(17).cuda()))
    assert not torch.equal(pam.dropout(x, 0.5, 17), pam.dropout(x, 0.5, 18))
    torch.manual_seed(5)
    a, b = pam.dropout(x, 0.5), pam.dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(a, pam.dropout(x, 0.5)) and not torch.equal(a, b)
    with pytest.raises(RuntimeError):
        pam.dropout(x, 0.5, torch.tensor([17]))


def test_share_that_stays(pam):
    # n = 2^22 draws: four standard deviations of a share are 4 sqrt(p (1 - p) / n) <= 2^-10
    for p in (0.1, 0.5, 0.73):
        out = pam.dropout(torch.ones(1 << 22).cuda(), p, 8)
        assert abs(float((out != 0).double().mean()) - (1 - p)) < 2 ** -10


def test_dropped_places_are_not_looked_at(pam):
    x = torch.full((4096,), float("nan"))
    _, mask = define.dropped(x, 0.5, 21)
    x[mask] = 1.5
    x[~mask] = torch.tensor([float("nan"), float("inf"), float("-inf")]).repeat(4096)[:int((~mask).sum())]
    out = pam.dropout(x.cuda(), 0.5, 21)
    assert bool(out.isfinite().all()) and torch.equal(out.cpu() != 0, mask)


def test_offset(pam):
    x = data(500, 6).cuda()
    kept = pam.dropout(torch.ones(500).cuda(), 0.2, 4) != 0
    assert torch.equal(pam.dropout(x, 0.2, 4, offset=1.0625), torch.where(kept, pam.mul(x, define.scale_of(0.2), offset=1.0625), 0.0))


def test_empty(pam):
    x = torch.zeros(0, 5, requires_grad=True, device="cuda")
    out = pam.dropout(x, 0.5, residual=x)
    out.sum().backward()
    assert out.shape == (0, 5) and x.grad.shape == (0, 5)


def test_far_elements(pam):
    """Places beyond 2^31 have counters of their own."""
    n = 2 ** 31 + 4099
    out = pam.dropout(torch.ones(n, device="cuda"), 0.5, 77)
    for first in (2 ** 31 - 50, n - 101):
        want = torch.where(define.kept(77, first, first + 101, 0.5), 2.0, 0.0)
        assert torch.equal(out[first:first + 101].cpu(), want)


def test_captured_with_new_masks(pam):
    """A captured forward and backward pass draws another mask at each replay, the same one both ways."""
    drop = pam.Dropout(0.5, approx_bwd=True)
    x = torch.ones(2000, device="cuda").requires_grad_()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(drop(x).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = drop(x)
        (dx,) = torch.autograd.grad(out.sum(), x)
    seen = []
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, dx)
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_seed_is_kept_for_the_backward_pass(pam):
    x = torch.ones(100, device="cuda").requires_grad_()
    seed = torch.tensor([3], device="cuda")
    out = pam.dropout(x, 0.5, seed, approx_bwd=True)
    seed += 1
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_no_second_derivative(pam):
    x = torch.ones(8, device="cuda").requires_grad_()
    (d,) = torch.autograd.grad(pam.dropout(x, 0.5, 1).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
