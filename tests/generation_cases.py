"""Beam search without caches: every step runs the decoder over the whole hypothesis, one after another."""
import torch

CONFIG = dict(vocab=40, dim=32, ffn=48, heads=4, encoder_layers=2, decoder_layers=2)
INF = float("inf")


def model(cfgs, device, seed=0):
    from pam_b200 import models, steps
    cfg = steps.TransformerConfig(**CONFIG)
    net = models.Transformer(cfg, **cfgs)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, p in net.named_parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (0.6 * p.shape[-1] ** -0.5 if p.dim() > 1 else 0.1) + (1.0 if "norm.weight" in name else 0.0))
    return net.to(device)


@torch.no_grad()
def search(net, src, beam, max_len, min_len, length_penalty, log_softmax, eos=2):
    """For one sentence [1, length]: [(score, tokens)], best first."""
    pad, live, done = net.cfg.pad, [(0.0, [])], []
    for t in range(max_len):
        found = []
        for b, (score, tokens) in enumerate(live):
            prev = torch.tensor([[eos] + tokens], device=src.device)
            lprobs = log_softmax(net(src, prev)[0, -1]).double().cpu()
            for token in range(net.cfg.vocab):
                allowed = token == eos if t == max_len - 1 else token != pad and (token != eos or t + 1 >= min_len)
                if allowed:
                    found.append((score + float(lprobs[token]), b, token))
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        done += [(s / (t + 1) ** length_penalty, live[b][1] + [token]) for s, b, token in found[:beam] if token == eos]
        live = [(s, live[b][1] + [token]) for s, b, token in found[:2 * beam] if token != eos][:beam]
        if len(done) >= beam:
            break
    done.sort(key=lambda h: -h[0])
    return done[:beam]


@torch.no_grad()
def rescored(net, src, tokens, length_penalty, log_softmax, eos=2):
    """The score of one hypothesis from the decoder over all of it at once."""
    prev = torch.tensor([[eos] + tokens[:-1]], device=src.device)
    lprobs = torch.stack([log_softmax(x) for x in net(src, prev)[0]]).double().cpu()
    return float(lprobs[torch.arange(len(tokens)), torch.tensor(tokens)].sum()) / len(tokens) ** length_penalty


def check(net, src, lengths, beam, max_len, min_len, length_penalty, log_softmax, tolerance, eos=2):
    """Each hypothesis has the score that the decoder gives it, and there are no worse ones than the search without caches finds (candidates
    within the tolerance of each other may change places)."""
    tokens, scores = net.generate(src, beam, max_len, src_lengths=lengths, min_len=min_len, length_penalty=length_penalty)
    assert tokens.shape[:2] == scores.shape == (src.shape[0], beam) and tokens.shape[2] <= max_len
    for g in range(src.shape[0]):
        n = src.shape[1] if lengths is None else int(lengths[g])
        want = search(net, src[g:g + 1, :n], beam, max_len, min_len, length_penalty, log_softmax)
        found = [(float(s), t[t != net.cfg.pad].tolist()) for s, t in zip(scores[g], tokens[g]) if float(s) > -INF]
        assert len(found) >= len(want) and len({tuple(t) for _, t in found}) == len(found)
        assert [s for s, _ in found] == sorted((s for s, _ in found), reverse=True)
        for score, t in found:
            assert t[-1] == eos and eos not in t[:-1] and min_len <= len(t) <= max_len
            assert abs(score - rescored(net, src[g:g + 1, :n], t, length_penalty, log_softmax)) <= tolerance
        for (a, _), (b, _) in zip(found, want):
            # (sentences of a batch go on until the last one is done: those that were done first may find better hypotheses)
            assert a >= b - tolerance and (src.shape[0] > 1 or a <= b + tolerance)
