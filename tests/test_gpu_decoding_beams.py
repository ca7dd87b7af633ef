"""beam_select and reorder_states against their definitions."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
INF = float("inf")


def _check(logits, scores, k, banned=None):
    from pam_b200 import decoding
    got = decoding.beam_select(logits, scores, k, banned)
    want = oracle.select(logits.cpu(), scores.cpu(), k, None if banned is None else banned.cpu())
    assert [tuple(t.shape) for t in got] == [(logits.shape[0], k)] * 3
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    best = got[0].double().cpu()
    low = want[0] == -INF
    assert bool((best[low] == -INF).all())
    assert bool(((best[~low] - want[0][~low]).abs() <= oracle.select_bound(want[0][~low])).all())
    return got


def _inputs(seed, groups, beams, vocab, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(groups, beams, vocab, generator=g).to(DEV) * scale, (-3 * torch.rand(groups, beams, generator=g)).to(DEV), g)


@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 1, 3), (2, 3, 2, 6), (3, 5, 100, 10), (1, 2, 31, 40), (4, 1, 4092, 3), (2, 2, 4093, 4), (2, 4, 4096, 8),
    (1, 3, 8185, 6), (2, 5, 10000, 10), (1, 4, 33001, 8), (1, 2, 151643, 4), (5, 16, 999, 32), (2, 20, 500, 64), (1, 64, 300, 64), (70, 5, 77, 10),
    (1, 33, 4500, 33),
])
def test_against_the_definition(groups, beams, vocab, k):
    logits, scores, _ = _inputs(vocab + k, groups, beams, vocab)
    _check(logits, scores, k)


def test_first_step_and_dead_beams():
    logits, scores, _ = _inputs(1, 3, 4, 500)
    logits[0, 1] = float("nan")                             # (not read)
    scores[0, 1:] = -INF
    scores[1, 2] = float("nan")
    scores[2] = -INF                                        # nothing goes on: the first tokens of the first beam
    best, beams, tokens = _check(logits, scores, 8)
    assert bool((beams[0] == 0).all()) and beams[2].tolist() == [0] * 8 and tokens[2].tolist() == list(range(8))


def test_fewer_live_candidates_than_asked_for():
    logits, scores, _ = _inputs(2, 2, 3, 6)
    scores[:, 1] = -INF
    logits[0, 0, 2:] = -INF
    logits[:, 2, 1:4] = torch.finfo(torch.float32).min
    _check(logits, scores, 18)


@pytest.mark.parametrize("value", [float("nan"), INF, 1e37, -INF, -1e30, torch.finfo(torch.float32).min, 0.0, -0.0, 1e-40, -9e29, 1e30])
def test_special_logits(value):
    logits, scores, _ = _inputs(3, 2, 3, 5000)
    logits[0, 1, 7] = value
    logits[1, 0, 3::5] = value
    logits[1, 2] = value
    _check(logits, scores, 9)


def test_special_logits_under_a_ban():
    """Banned tokens keep their share, whatever it is; masked ones have none."""
    logits, scores, g = _inputs(4, 2, 3, 700)
    banned = torch.rand(2, 3, 700, generator=g).to(DEV) < 0.3
    logits[0, 1][banned[0, 1]] = -INF
    logits[1, 1][banned[1, 1]] = float("nan")
    _check(logits, scores, 6, banned)


@pytest.mark.parametrize("shape", ["vocab", "group", "beam", "strided"])
def test_banned_tokens(shape):
    logits, scores, g = _inputs(5, 3, 4, 9001)
    flags = torch.rand(3, 4, 9001, generator=g).to(DEV) < 0.5
    banned = {"vocab": flags[0, 0], "group": flags[:, :1], "beam": flags, "strided": flags.transpose(1, 2).contiguous().transpose(1, 2)}[shape]
    _check(logits, scores, 8, banned)


def test_all_banned_but_a_few():
    logits, scores, _ = _inputs(6, 2, 5, 10000)
    banned = torch.ones(10000, dtype=torch.bool, device=DEV)
    _check(logits, scores, 10, banned)
    banned[[3, 9999, 5000]] = False
    _check(logits, scores, 10, banned)
    _check(logits, scores, 64, banned)


@pytest.mark.parametrize("k", [1, 10, 32, 33, 64])
def test_ties(k):
    """Equal logits, equal beams, equal everything: the lower beam, then the lower token."""
    logits, scores, _ = _inputs(7, 3, 5, 9000)
    logits = torch.round(logits)
    logits[1] = logits[1, :1]
    scores[1] = scores[1, 0]
    logits[2] = 0.25
    scores[2] = -1.0
    _check(logits, scores, k)


def test_steep_and_flat_logits():
    for scale in (1e-6, 0.01, 30.0, 1e4):
        logits, scores, _ = _inputs(8, 2, 4, 6000, scale)
        _check(logits, scores, 8)


def test_matches_log_softmax():
    import pam_b200 as pam
    logits, scores, _ = _inputs(10, 2, 3, 800)
    from pam_b200 import decoding
    best, beams, tokens = decoding.beam_select(logits, scores, 6)
    lprobs = pam.log_softmax(logits, dim=-1) + scores.unsqueeze(-1)
    chosen = lprobs[torch.arange(2, device=DEV)[:, None], beams, tokens]
    # (fp32 shift + log2, their division, two sums: four roundings at magnitudes below 16, and the sum of 800 terms)
    assert bool(((best - chosen).abs() <= (4 * 16 + 2 * 800) * oracle.U).all())


def test_layouts():
    logits, scores, _ = _inputs(11, 3, 4, 1003)
    want = _check(logits, scores, 8)
    from pam_b200 import decoding
    padded = torch.full((3, 4, 1024), float("nan"), device=DEV)
    for start in (0, 1, 2, 3):
        view = padded[:, :, start:start + 1003]
        view.copy_(logits)
        for a, b in zip(decoding.beam_select(view, scores, 8), want):
            assert torch.equal(a, b)
    for view in (logits.transpose(0, 1).contiguous().transpose(0, 1), logits.transpose(1, 2).contiguous().transpose(1, 2)):
        for a, b in zip(decoding.beam_select(view, scores.t().contiguous().t(), 8), want):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    step = (1 << 31) + 12
    buffer = torch.empty(2 * step + 4096, device=DEV)
    logits, scores, _ = _inputs(12, 3, 1, 2000)
    far = buffer.as_strided((3, 1, 2000), (step, step, 1))
    far.copy_(logits)
    _check(far, scores, 5)


def test_select_captured():
    from pam_b200 import decoding
    logits, scores, _ = _inputs(13, 3, 5, 10000)
    want = decoding.beam_select(logits, scores, 10)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decoding.beam_select(logits, scores, 10)
    for _ in range(3):
        for t in out:
            t.fill_(3)
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


# ---- reordering --------------------------------------------------------------------------------------------

def _moved(states, parents, used=None):
    out = []
    for t in states:
        new = t.clone()
        for g in range(parents.shape[0]):
            for r in range(parents.shape[1]):
                p = int(parents[g, r])
                if 0 <= p < parents.shape[1]:
                    if used is None:
                        new[g, r] = t[g, p]
                    else:
                        new[g, r, :used] = t[g, p, :used]
        out.append(new)
    return out


def _states(seed, groups, rows):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g).to(DEV)
    return [randn(groups, rows, 9, 4, 16), randn(groups, rows, 9, 3), randn(groups, rows, 70, 33), randn(groups, rows, 5, 8).half(),
            torch.randint(0, 1000, (groups, rows, 12), generator=g).to(DEV), torch.randint(0, 2, (groups, rows, 7), generator=g).bool().to(DEV),
            randn(groups, rows, 1, 1), torch.randint(0, 255, (groups, rows, 33, 5), generator=g).to(torch.uint8).to(DEV)], g


@pytest.mark.parametrize("groups,rows", [(1, 1), (3, 2), (2, 4), (3, 5), (1, 8), (2, 13), (1, 16), (2, 17), (1, 64)])
@pytest.mark.parametrize("used", [None, 0, 1, 5])
def test_reorder(groups, rows, used):
    from pam_b200 import decoding
    states, g = _states(groups + rows, groups, rows)
    if used == 5:
        states = [t for t in states if t.shape[2] >= 5]
    elif used == 1:
        states.append(torch.randn(groups, rows, 1, generator=g).to(DEV))
    for kind in range(3):
        parents = (torch.randint(0, rows, (groups, rows), generator=g) if kind < 2 else torch.randint(-2, rows + 2, (groups, rows), generator=g)).to(DEV)
        want = _moved(states, parents, used)
        versions = [t._version for t in states]
        decoding.reorder_states(states, parents, used)
        for a, b in zip(states, want):
            assert torch.equal(a, b)
        if used != 0:
            assert all(t._version > v for t, v in zip(states, versions))


def test_reorder_counts_on_the_device():
    from pam_b200 import decoding
    states, g = _states(3, 2, 5)
    for used in (0, 1, 4, 9, 1000, -4):
        parents = torch.randint(0, 5, (2, 5), generator=g).to(DEV)
        want = [_moved([t], parents, min(max(used, 0), t.shape[2]))[0] for t in states]
        decoding.reorder_states(states, parents, torch.tensor([used], device=DEV))
        for a, b in zip(states, want):
            assert torch.equal(a, b)


def test_reorder_views():
    """Rows of larger buffers: what lies between and behind them stays as it was."""
    from pam_b200 import decoding
    g = torch.Generator().manual_seed(4)
    buffer = torch.randn(3, 6, 2, 20, 40, generator=g).to(DEV)
    parents = torch.randint(0, 5, (3, 5), generator=g).to(DEV)
    before = buffer.clone()
    views = [buffer[:, 1:, 0], buffer[:, 1:, 1]]
    want = _moved(views, parents, 7)
    decoding.reorder_states(views, parents, 7)
    for a, b in zip(views, want):
        assert torch.equal(a, b)
    assert torch.equal(buffer[:, 0], before[:, 0]) and torch.equal(buffer[:, :, :, 7:], before[:, :, :, 7:])
    turned = torch.randn(5, 3, 11, generator=g).to(DEV).transpose(0, 1)
    want = _moved([turned], parents)
    decoding.reorder_states([turned], parents)
    assert torch.equal(turned, want[0])
    odd = torch.randn(3 * 5 * 8 + 1, generator=g).to(DEV)[1:].view(3, 5, 8)
    want = _moved([odd], parents)
    decoding.reorder_states([odd], parents)
    assert torch.equal(odd, want[0])


def test_reorder_many_tensors():
    from pam_b200 import decoding
    g = torch.Generator().manual_seed(5)
    states = [torch.randn(2, 3, 1 + i % 7, 4, generator=g).to(DEV) for i in range(300)]
    parents = torch.tensor([[2, 0, 1], [1, 1, 0]], device=DEV)
    want = _moved(states, parents)
    decoding.reorder_states(states, parents)
    for a, b in zip(states, want):
        assert torch.equal(a, b)


def test_reorder_beyond_32_bits():
    from pam_b200 import decoding
    step = 1 << 31
    buffer = torch.empty(2 * step + 64, device=DEV)
    state = buffer.as_strided((1, 3, 8, 4), (3 * step, step, 4, 1))
    state.copy_(torch.randn(1, 3, 8, 4))
    parents = torch.tensor([[2, 0, 0]], device=DEV)
    want = _moved([state.contiguous()], parents)
    decoding.reorder_states([state], parents)
    assert torch.equal(state, want[0])


def test_reorder_captured():
    from pam_b200 import decoding
    states, g = _states(6, 2, 5)
    parents, used = torch.tensor([[1, 2, 3, 4, 0], [0, 0, 4, 4, 1]], device=DEV), torch.tensor([3], device=DEV)
    keep = [t.clone() for t in states]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        decoding.reorder_states(states, parents, used)
    for a, b in zip(states, keep):
        a.copy_(b)
    want = keep
    for n in (3, 0, 9):
        used.fill_(n)
        want = [_moved([t], parents, min(n, t.shape[2]))[0] for t in want]
        graph.replay()
        for a, b in zip(states, want):
            assert torch.equal(a, b)
