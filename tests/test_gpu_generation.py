"""Beam search of the translation model in PAM arithmetic: attention over caches, selection and reordering together."""
import pytest
import torch

import generation_cases as cases

pytestmark = pytest.mark.gpu


def _net(seed=0, **settings):
    import json
    dkw = dict(approx_bwd=True, **settings)
    cfgs = dict(linear_cfg=json.dumps({"subtype": "pam", "dkwargs": dkw}), norm_cfg=json.dumps({"subtype": "pam_ln", "dkwargs": dkw}),
                functional_cfg=json.dumps({"type": "pam", "dkwargs": dkw}))
    return cases.model(cfgs, "cuda", seed)


def _log_softmax():
    import pam_b200 as pam
    return lambda x: pam.log_softmax(x.unsqueeze(0), dim=-1)[0]


# Scores near -10 are sums of up to eight log-probabilities.  Whole sequences and single tokens add the same products in other orders and shift the
# softmax by other whole numbers; piecewise affine functions have slopes of at most 2 each, so a few hundred roundings of 2^-24
# at magnitudes up to 16 come to a few 1e-4 at the very most.
TOLERANCE = 1e-3


@pytest.mark.parametrize("beam,max_len,min_len,penalty", [(1, 6, 1, 1.0), (3, 8, 1, 1.0), (5, 7, 4, 0.6), (2, 1, 1, 1.0), (9, 5, 1, 1.0)])
def test_against_search_without_caches(beam, max_len, min_len, penalty):
    net = _net()
    src = torch.randint(4, net.cfg.vocab, (3, 7), generator=torch.Generator().manual_seed(beam)).cuda()
    for g in range(3):
        cases.check(net, src[g:g + 1], None, beam, max_len, min_len, penalty, _log_softmax(), TOLERANCE)
    cases.check(net, src, None, beam, max_len, min_len, penalty, _log_softmax(), TOLERANCE)


def test_padded_batch():
    net = _net(1)
    src = torch.randint(4, net.cfg.vocab, (3, 9), generator=torch.Generator().manual_seed(3)).cuda()
    lengths = torch.tensor([9, 4, 6], device="cuda")
    cases.check(net, src, lengths, 3, 8, 1, 1.0, _log_softmax(), TOLERANCE)
    other = src.clone()
    other[1, 4:], other[2, 6:] = 1, 5
    got, want = net.generate(src, 3, 8, src_lengths=lengths), net.generate(other, 3, 8, src_lengths=lengths)
    # (the encoder's softmax shifts by the whole tensor's maximum, the padding's queries among it: the same up to rounding)
    assert bool(((got[1] - want[1]).abs() <= TOLERANCE).all())


def test_an_offset_takes_the_operator_dictionary(monkeypatch):
    """With an offset the softmax depends on the whole tensor's maximum: the dictionary's functions run as they stand."""
    from pam_b200 import decoding
    for name in ("cached_attention", "beam_select"):
        monkeypatch.setattr(decoding, name, None)
    net = _net(1, offset=1.02)
    tokens, scores = net.generate(torch.full((2, 5), 7, device="cuda"), 3, 6, src_lengths=torch.tensor([5, 3], device="cuda"))
    assert bool(scores.isfinite().all()) and bool((tokens == 2).any(-1).all())


def test_uses_the_operators(monkeypatch):
    from pam_b200 import decoding
    calls = {}
    for name in ("cached_attention", "beam_select", "reorder_states"):
        def counted(*a, _real=getattr(decoding, name), _name=name, **kw):
            calls[_name] = calls.get(_name, 0) + 1
            return _real(*a, **kw)
        monkeypatch.setattr(decoding, name, counted)
    net = _net(2)
    net.generate(torch.full((2, 5), 7, device="cuda"), 4, 6, min_len=6)
    assert calls["beam_select"] == 6 and calls["cached_attention"] == 6 * 4 and calls["reorder_states"] == 5 * 2


def test_on_another_stream():
    net = _net(3)
    src = torch.randint(4, net.cfg.vocab, (4, 9)).cuda()
    want = net.generate(src, 4, 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = net.generate(src, 4, 8)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_training_goes_on_after_generation():
    net = _net(4)
    src = torch.randint(4, net.cfg.vocab, (2, 6)).cuda()
    before = net(src, src).detach()
    net.generate(src, 3, 5)
    out = net(src, src)
    assert torch.equal(out, before)
    out.sum().backward()
    assert all(p.grad is not None for p in net.parameters())
