"""Sampling from the translation model where rows of logits leave no token to draw, on the CPU."""
import pytest
import torch

import generation_cases as cases

INF = float("inf")


def test_rows_without_a_token_end(monkeypatch):
    from pam_b200 import models
    net = cases.model({}, "cpu")
    src = torch.randint(4, net.cfg.vocab, (2, 6), generator=torch.Generator().manual_seed(1))
    draw, step, fed = models._draw, models.Transformer._step, []

    def drawn(*a):
        tokens, scores = draw(*a)
        if len(fed) == 3:                                     # the third tokens of two samples
            tokens[0, 1] = tokens[1, 0] = -1
            scores[0, 1] = scores[1, 0] = -INF
        return tokens, scores

    def stepped(self, last, *a):
        fed.append(last.clone())
        return step(self, last, *a)
    sample = lambda: net.sample(src, 3, 6, min_len=6, generator=torch.Generator().manual_seed(5))
    want = sample()
    monkeypatch.setattr(models, "_draw", drawn)
    monkeypatch.setattr(models.Transformer, "_step", stepped)
    tokens, scores = sample()
    assert len(fed) == 6 and all(bool(((t >= 0) & (t < net.cfg.vocab)).all()) for t in fed)
    for g in range(2):
        for s in range(3):
            if (g, s) in ((0, 1), (1, 0)):
                assert torch.equal(tokens[g, s, :2], want[0][g, s, :2]) and bool((tokens[g, s, 2:] == net.cfg.pad).all()) and float(scores[g, s]) == -INF
            else:
                assert torch.equal(tokens[g, s], want[0][g, s]) and torch.equal(scores[g, s], want[1][g, s])


def test_nothing_to_draw_at_all(monkeypatch):
    from pam_b200 import models
    net = cases.model({}, "cpu")
    shape = lambda logits: (torch.full(logits.shape[:-1], -1), torch.full(logits.shape[:-1], -INF))
    monkeypatch.setattr(models, "_draw", lambda ops, logits, *a: shape(logits))
    tokens, scores = net.sample(torch.full((2, 4), 7), 3, 9)
    assert tokens.shape == (2, 3, 1) and bool((tokens == net.cfg.pad).all()) and bool((scores == -INF).all())


@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.7, 3, 0.8, 0.1)])
def test_draws_of_ordinary_operators(settings):
    """Rows with a NaN, and rows whose tokens are all banned or masked, have no token; the others theirs."""
    from pam_b200 import models
    ops = dict(div=torch.div, log_softmax=torch.log_softmax)
    logits = torch.randn(5, 12, generator=torch.Generator().manual_seed(2))
    u = torch.rand(5, generator=torch.Generator().manual_seed(3))
    banned = torch.zeros(12, dtype=torch.bool)
    banned[[1, 5]] = True
    want = models._draw(ops, logits, u, *settings, banned)
    assert bool((want[0] >= 0).all()) and not bool(banned[want[0]].any())
    logits[1, 4] = float("nan")
    logits[2, ~banned] = -INF
    logits[3] = INF
    tokens, scores = models._draw(ops, logits, u, *settings, banned)
    assert tokens.tolist() == [int(want[0][0]), -1, -1, -1, int(want[0][4])]
    assert scores.tolist() == [float(want[1][0]), -INF, -INF, -INF, float(want[1][4])]
