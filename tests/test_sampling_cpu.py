"""Sampling from the translation model with the ordinary operators, and the model's dropout, on the CPU."""
import pytest
import torch

import generation_cases as cases


def test_samples_have_their_scores():
    net = cases.model({}, "cpu")
    src = torch.randint(4, net.cfg.vocab, (3, 7), generator=torch.Generator().manual_seed(1))
    tokens, scores = net.sample(src, 4, 8, min_len=2, generator=torch.Generator().manual_seed(5))
    again = net.sample(src, 4, 8, min_len=2, generator=torch.Generator().manual_seed(5))
    assert torch.equal(tokens, again[0]) and torch.equal(scores, again[1])
    assert tokens.shape[:2] == scores.shape == (3, 4) and len({tuple(t.tolist()) for t in tokens.view(12, -1)}) > 3
    for g in range(3):
        for t, score in zip(tokens[g], scores[g]):
            t = t[t != net.cfg.pad].tolist()
            assert t[-1] == 2 and 2 not in t[:-1] and 2 <= len(t) <= 8
            # (sums of up to eight fp32 log-probabilities near -4)
            assert abs(float(score) - cases.rescored(net, src[g:g + 1], t, 0.0, lambda x: torch.log_softmax(x, -1))) < 1e-4


def test_best_token_each_time():
    net = cases.model({}, "cpu", 3)
    src = torch.randint(4, net.cfg.vocab, (3, 7), generator=torch.Generator().manual_seed(2))
    want = net.generate(src, 1, 9, length_penalty=0.0)
    for kw in (dict(top_k=1), dict(top_p=1e-6), dict(min_p=1.0)):
        tokens, scores = net.sample(src, 1, 9, **kw)
        n = max(tokens.shape[2], want[0].shape[2])
        pad = lambda t: torch.nn.functional.pad(t, (0, n - t.shape[2]), value=net.cfg.pad)
        assert torch.equal(pad(tokens), pad(want[0])) and torch.allclose(scores, want[1], atol=1e-4)


def test_refusals():
    net = cases.model({}, "cpu")
    src = torch.full((1, 3), 4)
    for kw in (dict(samples=0), dict(max_len=0), dict(min_len=5, max_len=4), dict(eos=1), dict(eos=40), dict(src_lengths=torch.tensor([4])), dict(temperature=0.0), dict(top_k=-1),
               dict(top_k=1.5), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=True)):
        with pytest.raises(ValueError):
            net.sample(src, **kw)
    with pytest.raises(TypeError):
        net.sample(src, temperature=torch.ones(1, 5))


def test_dropout_in_training_alone():
    from pam_b200 import models, steps
    cfg = steps.TransformerConfig(**cases.CONFIG)
    with pytest.raises(ValueError):
        models.Transformer(cfg, dropout=1.0)
    net = models.Transformer(cfg, dropout=0.3)
    plain = models.Transformer(cfg)
    plain.load_state_dict(net.state_dict())
    src, out = torch.full((2, 5), 7), torch.full((2, 4), 9)
    assert not torch.equal(net(src, out), net(src, out))
    # (generation does without, in training mode too)
    assert torch.equal(net.generate(src, 2, 4)[1], plain.generate(src, 2, 4)[1])
    net.eval()
    assert torch.equal(net(src, out), plain(src, out))
    net.train()
    net(src, out).sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in net.parameters())
