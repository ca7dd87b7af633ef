"""The translation model through the operators at both ends of its vocabulary: training with dropout, and sampling."""
import pytest
import torch

import generation_cases as cases
from test_gpu_generation import TOLERANCE, _log_softmax, _net

pytestmark = pytest.mark.gpu


def _dropping(p=0.25, approx=True):
    from pam_b200 import models, steps
    cfgs = models.pam_cfgs(approx_bwd=approx)
    torch.manual_seed(0)
    cfg = steps.TransformerConfig(**cases.CONFIG)
    return models.Transformer(cfg, linear_cfg=cfgs["linear"], norm_cfg=cfgs["norm"], functional_cfg=cfgs["function"], loss_functional_cfg=cfgs["function"],
                              dropout=p).cuda()


def _batch(net):
    g = torch.Generator().manual_seed(1)
    src, out, target = (torch.randint(4, net.cfg.vocab, (3, n), generator=g).cuda() for n in (6, 5, 5))
    return src, out, target


@pytest.mark.parametrize("approx", [True, False])
def test_training_step_is_the_chain_with_the_same_masks(monkeypatch, approx):
    """The step through the fused operators is, to the bit forward, the one whose embedding and additions run one operator after another."""
    import pam_b200 as pam
    net = _dropping(approx=approx)
    batch = _batch(net)

    def step():
        net.zero_grad()
        torch.manual_seed(7)
        loss = net.loss(*batch)
        loss.backward()
        return loss.detach(), {k: p.grad.clone() for k, p in net.named_parameters()}
    calls = []

    def chain_embedding(tokens, weight, scale, positions, padding_idx, *, p=0.0, seed=None, **kw):
        calls.append("embedding")
        x = pam.mul(scale, torch.nn.functional.embedding(tokens, weight, padding_idx), **kw) + positions
        return real_dropout(x, p, seed, **kw) if p else x

    def chain_dropout(x, p, seed, residual, **kw):
        calls.append("dropout")
        return residual + real_dropout(x, p, seed, **kw)
    got = step()
    from pam_b200 import models
    real_dropout = models.pam_ops.dropout
    monkeypatch.setattr(models.pam_ops, "embedding", chain_embedding)
    monkeypatch.setattr(models.pam_ops, "dropout", chain_dropout)
    want = step()
    assert calls.count("embedding") == 2 and calls.count("dropout") == 2 * 2 + 3 * 2
    assert torch.equal(got[0], want[0])
    for k, g in got[1].items():
        if "embed_tokens" in k:
            # (each of at most 33 terms and the output projection's part: sums in another order, 2^-24 of the magnitudes for each addition)
            assert bool(((g - want[1][k]).abs() <= 64 * 2.0 ** -24 * want[1][k].abs().max()).all())
        else:
            assert torch.equal(g, want[1][k]), k


def test_masks_follow_the_seed():
    net = _dropping()
    src, out, target = _batch(net)
    torch.manual_seed(1)
    a, b = net(src, out), net(src, out)
    torch.manual_seed(1)
    assert torch.equal(a, net(src, out)) and not torch.equal(a, b)
    net.eval()
    assert torch.equal(net(src, out), net(src, out))


def test_embedding_without_gradients_is_the_chain():
    net = _dropping(0.0)
    tokens = torch.randint(0, net.cfg.vocab, (3, 9)).cuda()
    want = net.encoder.embed(tokens)
    with torch.no_grad():
        assert torch.equal(net.encoder.embed(tokens), want)


def test_encoder_in_a_graph():
    """Forward and backward passes captured once: each replay has masks of its own, and gradients that go with them.  (The positions are given: the table of a
    model is made on the host.)"""
    net = _dropping()
    src, stack = _batch(net)[0], net.encoder
    positions = stack._positions(src.shape[1], src.device).clone()
    params = list(stack.parameters())

    def step():
        x = stack.embed(src, positions)
        for layer in stack.layers:
            x = layer(x)
        total = (x * x).sum() + x.sum()
        return total, torch.autograd.grad(total, params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total, grads = step()
    totals = []
    for _ in range(3):
        graph.replay()
        totals.append(grads[0].clone())
        assert all(bool(g.isfinite().all()) for g in grads)
    assert not torch.equal(totals[0], totals[1]) and not torch.equal(totals[1], totals[2])


def test_samples_have_their_scores():
    net = _net()
    src = torch.randint(4, net.cfg.vocab, (3, 7), generator=torch.Generator().manual_seed(1)).cuda()
    generator = lambda: torch.Generator("cuda").manual_seed(5)
    tokens, scores = net.sample(src, 4, 8, min_len=2, temperature=1.0, generator=generator())
    again = net.sample(src, 4, 8, min_len=2, temperature=1.0, generator=generator())
    assert torch.equal(tokens, again[0]) and torch.equal(scores, again[1])
    for g in range(3):
        for t, score in zip(tokens[g], scores[g]):
            t = t[t != net.cfg.pad].tolist()
            assert t[-1] == 2 and 2 not in t[:-1] and 2 <= len(t) <= 8
            assert abs(float(score) - cases.rescored(net, src[g:g + 1], t, 0.0, _log_softmax())) <= TOLERANCE


def test_best_token_each_time():
    net = _net(3)
    src = torch.randint(4, net.cfg.vocab, (3, 7), generator=torch.Generator().manual_seed(2)).cuda()
    want = net.generate(src, 1, 9, length_penalty=0.0)
    for kw in (dict(top_k=1), dict(top_p=1e-6), dict(min_p=1.0)):
        tokens, scores = net.sample(src, 1, 9, **kw)
        n = max(tokens.shape[2], want[0].shape[2])
        pad = lambda t: torch.nn.functional.pad(t, (0, n - t.shape[2]), value=net.cfg.pad)
        assert torch.equal(pad(tokens), pad(want[0])) and bool(((scores - want[1]).abs() <= TOLERANCE).all())


def test_uses_the_operators(monkeypatch):
    from pam_b200 import decoding, models
    calls = []
    for module, name in ((decoding, "sample"), (decoding, "cached_attention"), (models.pam_ops, "embedding")):
        def counted(*a, _real=getattr(module, name), _name=name, **kw):
            calls.append(_name)
            return _real(*a, **kw)
        monkeypatch.setattr(module, name, counted)
    net = _net(2)
    net.sample(torch.full((2, 5), 7, device="cuda"), 4, 6, min_len=6, top_k=10, top_p=0.9)
    assert calls.count("sample") == 6 and calls.count("cached_attention") == 6 * 4 and calls.count("embedding") == 7
