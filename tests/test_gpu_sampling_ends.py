"""Sampling from the translation model on the GPU where rows of logits leave no token to draw."""
import pytest
import torch

from test_gpu_generation import _net

pytestmark = pytest.mark.gpu
INF = float("inf")


def test_temperature_at_the_end_of_its_range():
    net = _net()
    tokens, scores = net.sample(torch.full((2, 5), 7, device="cuda"), 3, 6, temperature=2.0 ** -126)    # (quotients beyond the PAM range)
    assert tokens.shape == (2, 3, 1) and bool((tokens == net.cfg.pad).all()) and bool((scores == -INF).all())


def test_rows_of_a_batch_end_alone(monkeypatch):
    net = _net()
    src = torch.randint(4, net.cfg.vocab, (2, 6), generator=torch.Generator().manual_seed(1)).cuda()
    sample = lambda: net.sample(src, 3, 6, min_len=6, generator=torch.Generator("cuda").manual_seed(5))
    want, project, steps = sample(), net.decoder.output_projection.forward, []

    def projected(x):
        logits = project(x)
        steps.append(1)
        if len(steps) == 3:
            logits[0, 1, 20] = float("nan")
            logits[1, 2] = -INF
        return logits
    monkeypatch.setattr(net.decoder.output_projection, "forward", projected)
    tokens, scores = sample()
    for g in range(2):
        for s in range(3):
            if (g, s) in ((0, 1), (1, 2)):
                assert torch.equal(tokens[g, s, :2], want[0][g, s, :2]) and bool((tokens[g, s, 2:] == net.cfg.pad).all()) and float(scores[g, s]) == -INF
            else:
                assert torch.equal(tokens[g, s], want[0][g, s]) and torch.equal(scores[g, s], want[1][g, s])
