"""Sampling on the GPU against its definition: the same token always, the score to its derived bound."""
import math

import pytest
import torch

import vocabulary_cases as define

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(scope="module")
def sample():
    from pam_b200 import decoding
    return decoding.sample


def check(sample, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, banned=None):
    dev = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v
    tokens, scores = sample(x.cuda(), u.cuda(), temperature=dev(temperature), top_k=dev(top_k), top_p=dev(top_p), min_p=dev(min_p), banned=dev(banned))
    assert tokens.dtype == torch.int64 and tokens.shape == scores.shape == u.shape
    rows = x.reshape(-1, x.shape[-1])
    ban = None if banned is None else banned.expand(x.shape).reshape(rows.shape)
    of = lambda v, r: v.flatten()[r].item() if isinstance(v, torch.Tensor) else v
    for r in range(rows.shape[0]):
        token, score, bound = define.sampled(rows[r], u.flatten()[r], of(temperature, r), of(top_k, r), of(top_p, r), of(min_p, r), None if ban is None else ban[r])
        assert int(tokens.flatten()[r]) == token, (r, int(tokens.flatten()[r]), token)
        got = float(scores.flatten()[r])
        assert got == score or abs(got - score) <= bound, (r, got, score)
    return tokens, scores


def data(rows, vocab, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, vocab, generator=g) * spread, torch.rand(rows, generator=g)


SETTINGS = [dict(), dict(top_k=1), dict(top_k=10), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=50, top_p=0.8, temperature=0.7), dict(top_p=0.5, min_p=0.3, temperature=1.5),
            dict(top_k=3, min_p=1.0), dict(top_p=2.0 ** -24)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v:g}" for k, v in s.items()) or "all")
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (4, 31), (4, 32), (2, 33), (5, 1000), (3, 4095), (2, 8193), (1, 10000), (2, 32768), (1, 32769), (1, 65537), (1, 262144), (160, 300)])
def test_against_definition(sample, rows, vocab, settings):
    check(sample, *data(rows, vocab, seed=vocab), **settings)


@pytest.mark.parametrize("spread", [0.0, 1e-30, 1e-6, 0.1, 20.0, 300.0, 1e6, 1e12, 1e29])
def test_spreads(sample, spread):
    for settings in SETTINGS:
        check(sample, *data(3, 700, seed=3, spread=spread), **settings)


@pytest.mark.parametrize("rows, vocab", [(3, 1000), (2, 20000), (2, 70000)])
@pytest.mark.parametrize("levels", [1, 2, 7])
def test_ties(sample, rows, vocab, levels):
    """Equal logits by the hundred: those that stay have the lowest numbers."""
    g = torch.Generator().manual_seed(levels)
    x = torch.randint(0, levels, (rows, vocab), generator=g) * 0.75
    u = torch.rand(rows, generator=g)
    for settings in SETTINGS + [dict(top_k=vocab // 3), dict(top_k=vocab // 2, top_p=0.33), dict(top_k=vocab - 1), dict(top_k=vocab), dict(top_k=vocab + 5), dict(top_k=2 ** 40)]:
        check(sample, x, u, **settings)


def test_edges_of_the_uniform_number(sample):
    x, _ = data(6, 500, seed=9)
    u = torch.tensor([0.0, 2.0 ** -24, 1 - 2.0 ** -24, 0.5, 2.0 ** -30, 0.99999])
    for settings in SETTINGS:
        check(sample, x, u, **settings)
    # numbers outside [0, 1) are taken as the nearest within
    tokens, _ = sample(x.cuda(), torch.tensor([-1.0, 1.0, 7.0, INF, -INF, float("nan")]).cuda())
    want, _ = sample(x.cuda(), torch.tensor([0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0, 0.0]).cuda())
    assert torch.equal(tokens, want)


def test_masked_banned_and_spoilt_rows(sample):
    x, u = data(12, 300, seed=4)
    x[0, 10:] = -INF
    x[1] = -INF
    x[2, 5:] = -1e30
    x[3, 7] = float("nan")
    x[4, 7] = INF
    x[5, 7] = 3e37
    x[6, ::2] = -INF
    x[7, 0] = 90.0                                                # all but certain
    x[8, 0], x[8, 1] = 500.0, -500.0
    for banned in (None, torch.arange(300) == 0, torch.arange(300) < 299, torch.ones(300, dtype=torch.bool), torch.rand(12, 300) < 0.5,
                   (torch.rand(12, 1) < 0.5)):
        for settings in (dict(), dict(top_k=5), dict(top_p=0.7), dict(min_p=0.1, temperature=0.6)):
            tokens, scores = check(sample, x, u, banned=banned, **settings)
            assert tokens[[1, 3, 4, 5]].eq(-1).all() and scores[[1, 3, 4, 5]].eq(-INF).all()


def test_banned_tokens_far_above(sample):
    """What may be drawn lies octaves, or a whole range of numbers, below what may not."""
    x, u = data(7, 400, seed=14)
    x[:, 3] = torch.tensor([20.0, 40.0, 90.0, 1e3, 1e6, 1e9, 1e30])
    for settings in (dict(), dict(top_k=4), dict(top_p=0.6)):
        check(sample, x, u, banned=torch.arange(400) == 3, **settings)


def test_settings_of_each_row(sample):
    x, u = data(24, 900, seed=6)
    g = torch.Generator().manual_seed(8)
    temperature = 0.5 + torch.rand(24, generator=g)
    top_k = torch.randint(0, 40, (24,), generator=g)
    top_p = torch.where(torch.rand(24, generator=g) < 0.3, 1.0, 0.2 + 0.8 * torch.rand(24, generator=g))
    min_p = 0.2 * torch.rand(24, generator=g)
    check(sample, x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    check(sample, x, u, temperature=temperature, top_p=0.6)
    check(sample, x.view(4, 6, 900), u.view(4, 6), temperature=temperature.view(4, 6), top_k=top_k.view(4, 6), banned=torch.rand(6, 900) < 0.1)
    # out of range on the device
    bad = torch.tensor([0.0, -1.0, INF, float("nan")])
    tokens, scores = sample(x[:4].cuda(), u[:4].cuda(), temperature=bad.cuda())
    assert tokens.eq(-1).all() and scores.eq(-INF).all()
    plain = sample(x[:4].cuda(), u[:4].cuda())[0]
    assert torch.equal(plain, sample(x[:4].cuda(), u[:4].cuda(), top_k=torch.tensor([0, -5, 900, 2 ** 50]).cuda(), top_p=torch.tensor([1.0, 2.0, INF, float("nan")]).cuda(),
                                     min_p=torch.tensor([0.0, -1.0, -INF, float("nan")]).cuda())[0])
    best = sample(x[:4].cuda(), u[:4].cuda(), top_k=1)[0]
    assert torch.equal(best, sample(x[:4].cuda(), u[:4].cuda(), top_p=torch.tensor([0.0, -1.0, -INF, 1e-9]).cuda())[0])
    assert torch.equal(best, sample(x[:4].cuda(), u[:4].cuda(), min_p=torch.tensor([1.0, 2.0, INF, 1.5]).cuda())[0])


def test_layouts(sample):
    x, u = data(12, 1001, seed=5)
    want = sample(x.cuda(), u.cuda(), top_p=0.9)
    wide = torch.zeros(12, 1010).cuda()
    for view in (wide[:, 1:1002], wide[:, 9:], torch.zeros(1001, 12).cuda().t(), torch.zeros(2, 1001).cuda()[:1].expand(12, 1001)):
        if view.stride(0) == 0:
            got = sample(view, u.cuda(), top_p=0.9)
            assert torch.equal(got[0], sample(view.contiguous(), u.cuda(), top_p=0.9)[0])
            continue
        view.copy_(x)
        got = sample(view, u.cuda(), top_p=0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ub = torch.zeros(12, 3).cuda()
    ub[:, 1] = u.cuda()
    assert torch.equal(sample(x.cuda(), ub[:, 1], top_p=0.9)[0], want[0])


def test_none(sample):
    tokens, scores = sample(torch.zeros(0, 7).cuda(), torch.zeros(0).cuda())
    assert tokens.shape == scores.shape == (0,)


def test_shares(sample):
    """Many draws from one row come out as often as they should."""
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5]).cuda()
    n = 1 << 20
    u = (torch.arange(n) / n).cuda()
    tokens, _ = sample(x.expand(n, 5), u)
    t = define.pam(define.pad(x.cpu(), 1.0), define.LOG2E)
    p = torch.exp2(torch.floor(t)) * (1 + t - torch.floor(t))
    p = p / p.sum()
    # (an even grid of n numbers is off by at most one number at each of a token's two borders)
    assert bool(((tokens.cpu().bincount(minlength=5).double() / n - p).abs() <= 2.0 / n + 2.0 ** -22).all())


def test_captured(sample):
    x, u = (t.cuda() for t in data(9, 5000, seed=12))
    graph = torch.cuda.CUDAGraph()
    sample(x, u, top_p=0.9)
    with torch.cuda.graph(graph):
        tokens, scores = sample(x, u, top_k=40, top_p=0.9)
    for seed in (1, 2):
        y, v = data(9, 5000, seed=seed)
        x.copy_(y)
        u.copy_(v)
        graph.replay()
        want = sample(x, u, top_k=40, top_p=0.9)
        assert torch.equal(tokens, want[0]) and torch.equal(scores, want[1])


@pytest.mark.parametrize("temperature", [2.0 ** -126, 1e-30, 1e-6, 1e-3, 0.37, 100.0, 1e6, 1e30, 2.0 ** 127])
def test_temperatures(sample, temperature):
    x, u = data(5, 800, seed=21)
    for settings in (dict(), dict(top_k=7), dict(top_p=0.8)):
        check(sample, x, u, temperature=temperature, **settings)


@pytest.mark.parametrize("rows, vocab", [(5, 1003), (3, 4097), (2, 30001), (2, 50002)])
def test_flags_at_odd_addresses(sample, rows, vocab):
    x, u = data(rows, vocab, seed=vocab)
    g = torch.Generator().manual_seed(1)
    for share in (0.0005, 0.3):
        banned = torch.rand(rows, vocab, generator=g) < share
        for settings in (dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.7)):
            check(sample, x, u, banned=banned, **settings)
            check(sample, x, u, banned=banned[0], **settings)


def test_values_that_the_range_rule_cuts_off(sample):
    """Zeros and denormals, and quads in which one value is far from the others."""
    x, u = data(6, 600, seed=31)
    x[0] = 0.0
    x[1, ::3] = 0.0
    x[2, ::5] = 1e-40
    x[3, ::7] = -0.0
    x[4] *= 1e-37
    x[5, ::4] = -INF
    for settings in SETTINGS:
        check(sample, x, u, **settings)


def test_large_k(sample):
    """Cuts that no list holds."""
    for rows, vocab in ((2, 5000), (1, 60000)):
        x, u = data(rows, vocab, seed=rows)
        for k in (127, 128, 129, 256, 257, 600, 4000):
            check(sample, x, u, top_k=k)
            check(sample, x, u, top_k=k, top_p=0.8, min_p=1e-4)
