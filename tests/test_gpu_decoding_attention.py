"""cached_attention against its definition in 64 bits, at the sizes, layouts and values where it can go wrong."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _check(got, q, own_k=None, own_v=None, own_lengths=None, shared_k=None, shared_v=None, shared_lengths=None):
    cpu = [t.cpu() if isinstance(t, torch.Tensor) else t for t in (q, own_k, own_v, own_lengths, shared_k, shared_v, shared_lengths)]
    want, bound = oracle.attention(*cpu)
    got = got.double().cpu()
    assert got.shape == want.shape
    assert bool((got.isnan() == want.isnan()).all()), "NaN in other places"
    err, ok = (got - want).abs(), ~want.isnan()
    assert bool((err[ok] <= bound[ok]).all()), f"off by {float((err[ok] / bound[ok]).max()):.3g} times the bound"


def _inputs(seed, groups, rows, heads, kv_heads, dim, shared, own, ragged=False):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g).to(DEV)
    case = dict(q=randn(groups, rows, heads, dim) * dim ** -0.5)
    if shared:
        case.update(shared_k=randn(groups, shared, kv_heads, dim), shared_v=randn(groups, shared, kv_heads, dim))
        if ragged:
            case["shared_lengths"] = torch.randint(0, shared + 1, (groups,), generator=g).to(DEV)
    if own:
        case.update(own_k=randn(groups, rows, own, kv_heads, dim), own_v=randn(groups, rows, own, kv_heads, dim))
        if ragged:
            case["own_lengths"] = torch.randint(0, own + 1, (groups, rows), generator=g).to(DEV)
    return case


def _run(case):
    from pam_b200 import decoding
    return decoding.cached_attention(**case)


@pytest.mark.parametrize("groups,rows,heads,kv_heads,dim,shared,own,ragged", [
    (1, 1, 1, 1, 1, 1, 0, False), (1, 1, 1, 1, 4, 0, 1, False), (2, 3, 2, 2, 64, 33, 0, False), (2, 5, 4, 4, 128, 32, 0, True),
    (3, 5, 4, 4, 128, 0, 17, True), (2, 4, 3, 3, 64, 65, 9, True), (1, 8, 2, 1, 32, 129, 40, True), (2, 3, 8, 2, 128, 70, 31, True),
    (1, 2, 8, 1, 256, 130, 5, True), (1, 7, 6, 2, 80, 47, 22, True), (1, 9, 2, 2, 96, 64, 64, False), (1, 17, 1, 1, 20, 50, 3, True),
    (2, 3, 2, 1, 67, 40, 13, True), (1, 6, 2, 2, 250, 37, 0, True), (1, 2, 2, 2, 3, 100, 100, True), (1, 5, 1, 1, 36, 513, 0, False),
    (1, 1, 2, 2, 64, 0, 2049, False), (1, 3, 1, 1, 16, 1025, 511, False), (40, 5, 4, 4, 16, 12, 7, True), (1, 1, 48, 1, 8, 90, 0, False),
    (300, 1, 2, 2, 8, 0, 65, True), (1, 64, 1, 1, 12, 20, 2, True),
])
def test_against_the_definition(groups, rows, heads, kv_heads, dim, shared, own, ragged):
    case = _inputs(groups * 1000 + dim, groups, rows, heads, kv_heads, dim, shared, own, ragged)
    _check(_run(case), **case)


def test_matches_the_chain_on_whole_sequences():
    """The last token of fused.attention_heads: the softmax shift is the tensor's there."""
    from pam_b200 import fused
    case = _inputs(5, 3, 4, 2, 2, 32, 50, 0)
    q, k, v = case["q"], case["shared_k"], case["shared_v"]
    chain = fused.attention_heads(q.reshape(3, 4, 64), k.reshape(3, 50, 64), v.reshape(3, 50, 64), 2).view(3, 4, 2, 32)
    want, bound = oracle.attention(q.cpu(), None, None, None, k.cpu(), v.cpu(), None)
    # (both lie within the bound; the chain's t - m is rounded at the magnitude of the tensor's shift, below 2^3 here)
    assert bool(((_run(case) - chain).double().cpu().abs() <= 2 * bound + 64 * oracle.U * want.abs().amax()).all())


def test_lengths_zero_one_and_beyond_the_slots():
    case = _inputs(12, 4, 2, 2, 2, 64, 20, 6)
    case["shared_lengths"] = torch.tensor([0, 1, 20, 1000], device=DEV)
    case["own_lengths"] = torch.tensor([[0, 1], [0, 6], [-3, 2], [9, 0]], device=DEV)
    out = _run(case)
    _check(out, **case)
    assert bool((out[0, 0] == 0).all())                    # nothing to see


def test_lengths_as_numbers():
    case = _inputs(13, 2, 2, 2, 2, 32, 20, 9)
    for shared, own in ((20, 0), (0, 9), (7, 3), (0, 0), (1, 1)):
        kw = dict(case, shared_lengths=shared, own_lengths=own)
        _check(_run(kw), **kw)


def test_what_lies_beyond_the_lengths_is_not_read():
    case = _inputs(14, 3, 3, 2, 2, 64, 70, 21, True)
    want = _run(case)
    for k in ("shared_k", "shared_v"):
        for g in range(3):
            case[k][g, int(case["shared_lengths"][g]):] = float("nan")
    for k in ("own_k", "own_v"):
        for g in range(3):
            for r in range(3):
                case[k][g, r, int(case["own_lengths"][g, r]):] = float("inf")
    assert torch.equal(_run(case), want)


@pytest.mark.parametrize("where", ["q", "shared_k", "shared_v", "own_k", "own_v"])
@pytest.mark.parametrize("value", [0.0, -0.0, 1e-40, 1e-30, 1e25, -1e25, float("inf"), float("nan")])
def test_special_values(where, value):
    case = _inputs(15, 2, 3, 2, 2, 64, 40, 10)
    t = case[where]
    t.view(-1)[:: 97] = value
    _check(_run(case), **case)


def test_scores_at_minus_infinity():
    """Sums that overflow to -inf count as masked, as in the softmax."""
    case = _inputs(16, 1, 2, 1, 1, 64, 10, 0)
    case["q"].fill_(1.0)
    case["shared_k"][:, 2] = -9e36
    case["shared_k"][:, 5] = -9e36
    _check(_run(case), **case)
    case["shared_k"].fill_(-9e36)
    assert bool(_run(case).isnan().all())                  # every position masked: 0 / 0, as there


def test_peaked_rows():
    """Probabilities far below the largest, down to those that vanish."""
    case = _inputs(17, 2, 3, 2, 2, 64, 60, 20)
    case["q"] *= 200.0
    _check(_run(case), **case)


def test_layouts():
    """Heads before positions, fused buffers, odd addresses, shared groups: views of any kind."""
    case = _inputs(18, 2, 3, 2, 2, 64, 33, 12, True)
    want = _run(case)
    swapped = dict(case)
    for name in ("shared_k", "shared_v", "own_k", "own_v"):
        swapped[name] = case[name].transpose(-3, -2).contiguous().transpose(-3, -2)
    assert torch.equal(_run(swapped), want)
    fused = dict(case)
    both = torch.stack([case["own_k"], case["own_v"]], 3)                          # [groups, rows, slots, 2, heads, dim]
    fused["own_k"], fused["own_v"] = both.unbind(3)
    fused["q"] = torch.cat([case["q"]] * 3, 2)[:, :, 2:4]
    assert torch.equal(_run(fused), want)
    odd = dict(case)
    for name in ("q", "shared_k", "shared_v", "own_k", "own_v"):
        t = case[name]
        buffer = torch.empty(t.numel() + 1, device=DEV)
        odd[name] = buffer[1:].view(t.shape).copy_(t)
        _check(_run(odd), **odd)
    spread = dict(case, shared_k=case["shared_k"][:1].expand(2, -1, -1, -1), shared_v=case["shared_v"][:1].expand(2, -1, -1, -1))
    _check(_run(spread), **spread)
    last = dict(case, q=case["q"].transpose(-1, -2).contiguous().transpose(-1, -2))
    assert torch.equal(_run(last), want)


def test_offsets_beyond_32_bits():
    """Positions 2^25 floats apart: the last ones lie beyond 2^31 elements and 2^33 bytes."""
    slots, step = 70, 1 << 25
    buffer = torch.empty(slots * step, device=DEV)
    rows = buffer.as_strided((1, slots, 2, 64), (slots * step, step, 64, 1))
    values = buffer[1 << 20:].as_strided((1, slots, 2, 64), (slots * step, step, 64, 1))
    case = _inputs(19, 1, 3, 2, 2, 64, slots, 0)
    rows.copy_(case["shared_k"])
    values.copy_(case["shared_v"])
    assert torch.equal(_run(dict(case, shared_k=rows, shared_v=values)), _run(case))


def test_same_bits_every_time():
    case = _inputs(20, 2, 4, 2, 2, 64, 3000, 100, True)
    want = _run(case)
    for _ in range(5):
        assert torch.equal(_run(case), want)


def test_on_another_stream():
    case = _inputs(21, 2, 4, 2, 2, 128, 400, 30, True)
    want = _run(case)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _run(case)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


def test_captured_graphs_share_nothing():
    """Two graphs captured one after the other, replayed in turn and with new lengths."""
    cases = [_inputs(22 + i, 2, 3, 2, 2, 64, 900, 40, True) for i in range(2)]
    want = [_run(c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(c))
        graphs.append(graph)
    for i in (0, 1, 0, 1, 1):
        outs[i].fill_(7.0)
        graphs[i].replay()
        assert torch.equal(outs[i], want[i])
    cases[0]["shared_lengths"].fill_(3)
    cases[0]["own_lengths"].fill_(0)
    graphs[0].replay()
    graphs[1].replay()
    _check(outs[0], **cases[0])
    assert torch.equal(outs[1], want[1])


@pytest.mark.parametrize("own", [False, True])
def test_far_above_the_first_scores(own):
    """Sums of 2^70 and more, shifted by what came first, beside exponentials near 2^-126: those are probabilities of zero."""
    first, high, low = 1.0, 50.25, -96.25                  # t: 1.4, 64.8 (above its floor by less than 64) and -124.6 (below it by less than 126)
    t = [float(oracle.pam(s, oracle.LOG2E)) for s in (first, high, low)]
    assert 1 <= t[0] < 2 and 64 <= t[1] < 65 and -125 <= t[2] < -124
    position = torch.arange(1000)
    s = torch.where(position // 32 % 8 < 4, first, high)
    s[position % 32 == 5] = torch.where(position // 32 % 8 < 4, first, low)[position % 32 == 5]
    k = torch.zeros(1000, 8)
    k[:, 0] = s
    v = torch.randn(1000, 8, generator=torch.Generator().manual_seed(50))
    v[s == low] = 2.0 ** 60
    q = torch.zeros(1, 1, 1, 8, device=DEV)
    q[..., 0] = 1.0
    name = "own" if own else "shared"
    lead = (1, 1, 1000, 1, 8) if own else (1, 1000, 1, 8)
    case = {"q": q, f"{name}_k": k.view(lead).to(DEV), f"{name}_v": v.view(lead).to(DEV)}
    _check(_run(case), **case)
