"""Embedding with scale, positions and dropout on the GPU against its definition."""
import math

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


def data(shape, vocab, dim, positions, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = math.prod(shape)
    tokens = torch.exp(torch.rand(n, generator=g) * math.log(vocab)).long().clamp(max=vocab - 1).view(shape)
    weight = torch.randn(vocab, dim, generator=g)
    pos = None if positions is None else torch.randn(shape[-1] if positions == "table" else 1, dim, generator=g)
    return tokens, weight, pos, torch.randn(*shape, dim, generator=g)


SHAPES = [((1,), 1, 1), ((5,), 7, 3), ((2, 3), 10, 4), ((1, 5), 1000, 512), ((9, 33), 503, 30), ((4, 64), 100, 128), ((3, 2, 50), 2000, 257), ((70, 61), 4000, 64),
          ((33, 250), 40, 36), ((12001,), 300000, 20), ((40, 500), 3, 8), ((3000,), 1 << 22, 5)]


@pytest.mark.parametrize("scale, positions, p, padding", [(None, None, 0.0, None), (22.6, "table", 0.3, 1), (0.7, "one", 0.0, 0), (3.0, None, 0.1, None), (None, "table", 0.5, None)])
@pytest.mark.parametrize("shape, vocab, dim", SHAPES)
@pytest.mark.parametrize("approx", [True, False])
def test_against_definition(pam, shape, vocab, dim, scale, positions, p, padding, approx):
    if padding is not None and padding >= vocab:
        padding = None
    tokens, weight, pos, g = data(shape, vocab, dim, positions)
    w = weight.cuda().requires_grad_()
    e = None if pos is None else pos.cuda().requires_grad_()
    out = pam.embedding(tokens.cuda(), w, scale, e, padding, p=p, seed=5, approx_bwd=approx)
    x, y = define.embedded(tokens, weight, scale, pos, p, 5)
    # the sum is rounded once and taken here from its rounded value, from which on everything is exact
    assert_bits_equal(out, y.float())
    grads = torch.autograd.grad(out, [w] + ([e] if e is not None else []), g.cuda())
    d, bound, h = define.embedded_grad(g, tokens, weight, scale, pos, padding, p, 5, approx)
    assert bool(((grads[0].double().cpu() - d).abs() <= bound).all())
    if e is not None:
        terms = h.flatten(0, -2).view(-1, pos.shape[0], dim)
        n = terms.shape[0]
        assert bool(((grads[1].double().cpu() - terms.sum(0)).abs() <= n * U * terms.abs().sum(0)).all())


def test_gradient_against_differences(pam):
    """Where the PAM product has one slope, a step of a table's element changes the sum by the exact gradient."""
    weight = (1.0 + torch.arange(12).view(3, 4) / 64).cuda().requires_grad_()
    tokens = torch.tensor([[0, 2, 2], [2, 1, 0]]).cuda()
    total = lambda w: pam.embedding(tokens, w, 1.25, p=0.25, seed=9).double().sum()
    (d,) = torch.autograd.grad(total(weight), weight)
    h = 2.0 ** -12
    with torch.no_grad():
        for v in range(3):
            for c in range(4):
                step = torch.zeros(3, 4).cuda()
                step[v, c] = h
                assert float((total(weight + step) - total(weight)) / h) == float(d[v, c])


def test_fused_is_the_chain(pam):
    """One call is the same, to the bit, as the operators one after another with the same seed."""
    tokens, weight, pos, g = data((6, 40), 700, 64, "table")
    t, w, e = tokens.cuda(), weight.cuda().requires_grad_(), pos.cuda()
    a = pam.embedding(t, w, 8.0, e, p=0.2, seed=3, approx_bwd=True)
    chain = pam.mul(8.0, torch.nn.functional.embedding(t, w), approx_bwd=True) + e
    b = pam.dropout(chain, 0.2, 3, approx_bwd=True)
    assert torch.equal(a, b)
    da, db = (torch.autograd.grad(y, w, g.cuda())[0] for y in (a, b))
    _, bound, _ = define.embedded_grad(g, tokens, weight, 8.0, pos, None, 0.2, 3, True)
    assert bool(((da - db).abs().cpu() <= 2 * bound).all())


def test_layouts(pam):
    tokens, weight, pos, g = data((8, 30), 500, 64, "table")
    plain = pam.embedding(tokens.cuda(), weight.cuda(), 2.0, pos.cuda(), p=0.1, seed=1)
    wide = torch.zeros(500, 131).cuda()
    for at, table in ((0, wide[:, :64]), (1, wide[:, 1:65]), (0, torch.zeros(64, 500).cuda().t())):
        table.copy_(weight)
        table = table.detach().requires_grad_()
        longer = torch.zeros(30, 70).cuda()[:, 3:67].copy_(pos)
        out = pam.embedding(tokens.cuda().t().contiguous().t(), table, 2.0, longer, p=0.1, seed=1, approx_bwd=True)
        assert torch.equal(out, plain)
        (d,) = torch.autograd.grad(out, table, g.cuda())
        want, bound, _ = define.embedded_grad(g, tokens, weight, 2.0, pos, None, 0.1, 1, True)
        assert bool(((d.double().cpu() - want).abs() <= bound).all())
        (d,) = torch.autograd.grad(pam.embedding(tokens.cuda(), table, 2.0, longer, p=0.1, seed=1), table, g.cuda())
        want, bound, _ = define.embedded_grad(g, tokens, weight, 2.0, pos, None, 0.1, 1, False)
        assert bool(((d.double().cpu() - want).abs() <= bound).all())
    gt = torch.zeros(30, 8, 64).cuda().transpose(0, 1).copy_(g)                      # a gradient with other strides
    w = weight.cuda().requires_grad_()
    a, b = (torch.autograd.grad(pam.embedding(tokens.cuda(), w, 2.0, approx_bwd=True), w, x)[0] for x in (gt, g.cuda()))
    assert torch.equal(a, b)
    assert torch.equal(pam.embedding(tokens.int().cuda(), w, 2.0), pam.embedding(tokens.cuda(), w, 2.0))


def test_tokens_outside_the_table(pam):
    weight = torch.randn(10, 6).cuda().requires_grad_()
    tokens = torch.tensor([3, -1, 10, 2 ** 40, -2 ** 63, 9]).cuda()
    out = pam.embedding(tokens, weight, 2.0)
    assert bool(out[1:5].isnan().all()) and bool(out[[0, 5]].isfinite().all())
    (d,) = torch.autograd.grad(out, weight, torch.ones(6, 6).cuda())
    assert bool(d.isfinite().all()) and d.abs().sum(1).nonzero().flatten().tolist() == [3, 9]


def test_all_padding_and_none(pam):
    weight = torch.randn(10, 6).cuda().requires_grad_()
    for tokens in (torch.full((50, 3), 4).cuda(), torch.zeros(0, 3, dtype=torch.int64).cuda()):
        out = pam.embedding(tokens, weight, 2.0, torch.zeros(3, 6).cuda(), 4, p=0.1)
        (d,) = torch.autograd.grad(out, weight, torch.ones_like(out))
        assert not d.any()


@pytest.mark.parametrize("n, dim", [(60000, 64), (60000, 7), (300000, 4)])
def test_one_token_over_and_over(pam, n, dim):
    """Sums of as many terms as there are tokens, the same from run to run."""
    g = torch.Generator().manual_seed(2)
    tokens = torch.full((n,), 5)
    tokens[::1000] = torch.arange(n)[::1000] % 11
    weight, dy = torch.randn(11, dim, generator=g), torch.randn(n, dim, generator=g)
    w = weight.cuda().requires_grad_()
    run = lambda: torch.autograd.grad(pam.embedding(tokens.cuda(), w, 3.0, p=0.1, seed=2, approx_bwd=True), w, dy.cuda())[0]
    d, bound, _ = define.embedded_grad(dy, tokens, weight, 3.0, None, None, 0.1, 2, True)
    got = run()
    assert bool(((got.double().cpu() - d).abs() <= bound).all())
    for _ in range(3):
        assert torch.equal(run(), got)


@pytest.mark.parametrize("n, vocab", [(4095, 5000), (4096, 5000), (4097, 5000), (8192, 130), (8193, 130), (70000, 20000), (70001, 262145)])
def test_many_tokens(pam, n, vocab):
    tokens, weight, _, g = data((n,), vocab, 12, None, seed=n)
    w = weight.cuda().requires_grad_()
    (d,) = torch.autograd.grad(pam.embedding(tokens.cuda(), w, 1.5, padding_idx=0, approx_bwd=True), w, g.cuda())
    want, bound, _ = define.embedded_grad(g, tokens, weight, 1.5, None, 0, 0.0, 0, True)
    assert bool(((d.double().cpu() - want).abs() <= bound).all())
    again = torch.autograd.grad(pam.embedding(tokens.cuda(), w, 1.5, padding_idx=0, approx_bwd=True), w, g.cuda())[0]
    assert torch.equal(d, again)


def test_streams_and_captures(pam):
    """Calls on several streams, and captures replayed in turn, do not share scratch."""
    tokens, weight, pos, g = data((20, 300), 900, 48, "table")
    w, dy = weight.cuda().requires_grad_(), g.cuda()
    other = torch.randint(0, 900, (20, 300)).cuda()
    step = lambda t: torch.autograd.grad(pam.embedding(t, w, 2.0, pos.cuda(), p=0.2, seed=6, approx_bwd=True), w, dy)[0]
    tok = tokens.cuda()
    want = [step(tok), step(other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s, t in zip(streams, (tok, other)):
            with torch.cuda.stream(s):
                got.append(step(t))
    torch.cuda.synchronize()
    for i, d in enumerate(got):
        assert torch.equal(d, want[i % 2])
    pos_d = pos.cuda()
    graphs = []
    for t in (tok, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            d = torch.autograd.grad(pam.embedding(t, w, 2.0, pos_d, p=0.2, seed=6, approx_bwd=True), w, dy)[0]
        graphs.append((graph, d))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
        for (_, d), x in zip(graphs, want):
            assert torch.equal(d, x)


def test_module(pam):
    torch.manual_seed(0)
    layer = pam.Embedding(50, 16, padding_idx=1, scale=4.0, p=0.5, approx_bwd=True).cuda()
    tokens = torch.tensor([[3, 1, 7]]).cuda()
    out = layer(tokens, torch.ones(3, 16).cuda(), seed=4)
    assert torch.equal(out, pam.embedding(tokens, layer.weight, 4.0, torch.ones(3, 16).cuda(), 1, p=0.5, seed=4))
    out.sum().backward()
    assert not layer.weight.grad[1].any() and bool(layer.weight.grad[3].any())
    layer.eval()
    assert torch.equal(layer(tokens), pam.mul(4.0, torch.nn.functional.embedding(tokens, layer.weight)))


@pytest.mark.parametrize("n, vocab, dim", [(3, 5001, 7), (9000, 5001, 7), (20000, 300000, 9), (5, 1, 1), (8193, 3, 2)])
def test_fills_all_rows(pam, n, vocab, dim):
    """Rows without a token are zeros, whatever was in their memory, at any address of the gradient."""
    from pam_b200 import _lib
    handle = _lib.lib()
    tokens = torch.randint(0, vocab, (n,)).cuda()
    dy = torch.randn(n, dim).cuda()
    ws_bytes = handle.pamk_embedding_bwd_workspace_bytes(n, vocab, dim)
    ws = torch.full((ws_bytes,), 0xAB, dtype=torch.uint8, device="cuda")
    want = torch.zeros(vocab, dim, dtype=torch.float64, device="cuda").index_add_(0, tokens, dy.double())
    for shift in (0, 1):
        memory = torch.full((vocab * dim + 8,), float("nan"), device="cuda")
        dw = memory[shift:shift + vocab * dim]
        _lib.check(handle.pamk_embedding_bwd(tokens.data_ptr(), dy.data_ptr(), None, dw.data_ptr(), n, vocab, dim, dim, -1, 0, 0.0, 0.0, None, 0, 1.0, 1,
                                             ws.data_ptr(), ws_bytes, torch.cuda.current_stream().cuda_stream), "pamk_embedding_bwd")
        count = tokens.bincount(minlength=vocab).double()[:, None]
        size = torch.zeros_like(want).index_add_(0, tokens, dy.double().abs())
        assert bool(((dw.view(vocab, dim).double() - want).abs() <= count * U * size).all())
        assert bool(memory[:shift].isnan().all()) and bool(memory[shift + vocab * dim:].isnan().all())
    assert handle.pamk_embedding_bwd(tokens.data_ptr(), dy.data_ptr(), None, dw.data_ptr(), n, vocab, dim, dim, -1, 0, 0.0, 0.0, None, 0, 1.0, 1, ws.data_ptr(),
                                     ws_bytes - 1, None) == -4


@pytest.mark.parametrize("scale", [0.0, -3.0, 1e-30, 1e30, 1e-45, 3e38, 1.0])
@pytest.mark.parametrize("dim", [8, 7])
def test_scales(pam, scale, dim):
    """Scales and values at the ends of the range: the products and slopes of pam.mul, to the bit."""
    tokens = torch.tensor([0, 3, 2, 1, 0]).cuda()
    some = torch.tensor([0.0, -0.0, 1e-40, -3e-38, 2e-20, -1.5, 7e18, -2e37, 1e38, float("inf"), float("nan")])
    g = torch.Generator().manual_seed(3)
    weight = some[torch.randint(0, len(some), (4, dim), generator=g)].cuda().requires_grad_()
    dy = some[torch.randint(0, 8, (5, dim), generator=g)].cuda()
    for approx in (True, False):
        out = pam.embedding(tokens, weight, scale, approx_bwd=approx)
        rows = torch.nn.functional.embedding(tokens, weight).detach().requires_grad_()
        want = pam.mul(scale, rows, approx_bwd=approx)
        assert_bits_equal(out, want)
        (d,), (terms,) = torch.autograd.grad(out, weight, dy), torch.autograd.grad(want, rows, dy)
        for v in (1, 2, 3):                                   # (one term each)
            assert_bits_equal(d[v] + 0.0, terms[tokens == v][0] + 0.0)


@pytest.mark.parametrize("runs", [(5000,), (1, 16 * 33, 16 * 34 - 1, 16 * 34 + 1, 17, 16, 15, 2000), (32 * 24, 32 * 25 - 1, 32 * 33 + 5, 40000, 1, 32 * 34, 32 * 1057 + 31, 32 * 66, 3), (5, 1100000, 7, 99)])
@pytest.mark.parametrize("dim", [4, 5, 132])
def test_lengths_of_runs(pam, runs, dim):
    """Sums of whole numbers below 2^24, which are exact in any order."""
    order = torch.randperm(sum(runs), generator=torch.Generator().manual_seed(dim))
    tokens = torch.arange(len(runs)).repeat_interleave(torch.tensor(runs))[order]
    g = torch.randint(-3, 4, (len(tokens), dim), generator=torch.Generator().manual_seed(2)).float()
    w = torch.zeros(len(runs) + 2, dim, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(pam.embedding(tokens.cuda(), w), w, g.cuda())
    want = torch.zeros(len(runs) + 2, dim, dtype=torch.float64).index_add_(0, tokens, g.double())
    assert torch.equal(d.double().cpu(), want)


def test_millions_of_tokens(pam):
    """More tokens than there are tiles at their smallest: a tile is walked over in several steps."""
    n, vocab = 2_200_003, 5001
    tokens, weight, _, g = data((n,), vocab, 2, None, seed=9)
    w = weight.cuda().requires_grad_()
    (d,) = torch.autograd.grad(pam.embedding(tokens.cuda(), w, 1.5, padding_idx=3, approx_bwd=True), w, g.cuda())
    want, bound, _ = define.embedded_grad(g, tokens, weight, 1.5, None, 3, 0.0, 0, True)
    assert bool(((d.double().cpu() - want).abs() <= bound).all())


def test_residual_and_input_are_one_tensor(pam):
    x = torch.randn(300, device="cuda").requires_grad_()
    y = pam.dropout(x, 0.4, 8, x, approx_bwd=True)
    (d,) = torch.autograd.grad(y, x, torch.ones_like(x))
    kept = pam.dropout(torch.ones(300, device="cuda"), 0.4, 8)
    assert torch.equal(d, kept + 1.0)


def test_expanded_positions(pam):
    tokens = torch.randint(0, 20, (3, 6)).cuda()
    w, row = torch.randn(20, 16).cuda().requires_grad_(), torch.randn(16).cuda().requires_grad_()
    a = pam.embedding(tokens, w, 2.0, row.expand(6, 16), approx_bwd=True)
    b = pam.embedding(tokens, w, 2.0, row, approx_bwd=True)
    assert torch.equal(a, b)
    ga, gb = (torch.autograd.grad(y, row, torch.ones_like(y))[0] for y in (a, b))
    assert torch.equal(ga, gb)                                # (sums of 18 ones)
