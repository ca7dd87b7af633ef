"""The operators of pam_b200.decoding through the native host path and through the Python layer: the same bits, the same refusals; and several
calls at once."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    from pam_b200 import _lib
    if request.param == "python":
        monkeypatch.setattr(_lib, "host", lambda: None)
    return request.param


def _attention_case(seed, own=30, shared=900):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g).to(DEV)
    return dict(q=randn(2, 3, 4, 64) * 0.125, own_k=randn(2, 3, own, 2, 64), own_v=randn(2, 3, own, 2, 64), own_lengths=torch.randint(0, own + 1, (2, 3), generator=g).to(DEV),
                shared_k=randn(2, shared, 2, 64), shared_v=randn(2, shared, 2, 64), shared_lengths=torch.randint(0, shared + 1, (2,), generator=g).to(DEV))


def _select_case(seed, vocab=10000):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(3, 4, vocab, generator=g).to(DEV), -torch.rand(3, 4, generator=g).to(DEV), 8, (torch.rand(3, 1, vocab, generator=g) < 0.1).to(DEV)


def _states(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(2, 5, 9, 8, generator=g).to(DEV), torch.randint(0, 9, (2, 5, 11), generator=g).to(DEV)], torch.randint(0, 5, (2, 5), generator=g).to(DEV)


def test_both_routes_agree(monkeypatch):
    from pam_b200 import _lib, decoding
    results = []
    for python in (False, True):
        with monkeypatch.context() as m:
            if python:
                m.setattr(_lib, "host", lambda: None)
            out = [decoding.cached_attention(**_attention_case(1)), decoding.cached_attention(**_attention_case(2, own=7))]
            case = _attention_case(3)
            out.append(decoding.cached_attention(case["q"], case["own_k"], case["own_v"], 11))
            out.append(decoding.cached_attention(case["q"], shared_k=case["shared_k"], shared_v=case["shared_v"], shared_lengths=0))
            out += decoding.beam_select(*_select_case(4))
            out += decoding.beam_select(*_select_case(5)[:3])
            for used in (None, 4, torch.tensor([6], device=DEV)):
                states, parents = _states(6)
                decoding.reorder_states(states, parents, used)
                out += states
            results.append(out)
    assert len(results[0]) == len(results[1])
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_refusals(route):
    from pam_b200 import decoding
    case = _attention_case(1)
    for change, error in ((dict(q=case["q"].cpu()), RuntimeError), (dict(shared_k=case["shared_k"].cpu()), RuntimeError), (dict(own_lengths=case["own_lengths"].cpu()), RuntimeError),
                          (dict(own_lengths=31), ValueError), (dict(own_lengths=-1), ValueError), (dict(own_lengths=case["own_lengths"].int()), ValueError),
                          (dict(own_k=case["own_k"].double(), own_v=case["own_v"].double()), TypeError), (dict(own_v=None), ValueError),
                          (dict(shared_v=case["shared_v"][:, :-1]), ValueError), (dict(q=case["q"][..., :32]), ValueError),
                          (dict(q=case["q"].detach().requires_grad_()), RuntimeError), (dict(own_k=case["own_k"].detach().requires_grad_()), RuntimeError)):
        with pytest.raises(error):
            decoding.cached_attention(**{**case, **change})
    logits, scores, k, banned = _select_case(1)
    for args, error in (((logits.cpu(), scores, k), RuntimeError), ((logits, scores.cpu(), k), RuntimeError), ((logits, scores, k, banned.cpu()), RuntimeError),
                        ((logits, scores, 65), ValueError), ((logits, scores[:, :2], k), ValueError), ((logits, scores, k, banned.float()), TypeError),
                        ((logits, scores, k, banned[:, :, :-1]), RuntimeError), ((logits.half(), scores, k), TypeError), ((logits.detach().requires_grad_(), scores, k), RuntimeError)):
        with pytest.raises(error):
            decoding.beam_select(*args)
    states, parents = _states(1)
    for args, error in ((([states[0], states[0]], parents), ValueError), (([states[0], states[0][:, :, 2:]], parents, 3), ValueError), ((states, parents.cpu()), RuntimeError),
                        ((states, parents, 10), ValueError), (([states[0].cpu()], parents), RuntimeError), ((states, parents, torch.tensor([1])), RuntimeError),
                        (([parents.unsqueeze(-1)], parents), ValueError), (([states[0].detach().requires_grad_()], parents), RuntimeError)):
        with pytest.raises(error):
            decoding.reorder_states(*args)


def test_without_grad_mode(route):
    from pam_b200 import decoding
    case = _attention_case(7)
    want = decoding.cached_attention(**case)
    case["q"].requires_grad_()
    with torch.no_grad():
        out = decoding.cached_attention(**case)
    assert not out.requires_grad and torch.equal(out, want)


def test_empty_calls(route):
    from pam_b200 import decoding
    z = lambda *shape: torch.zeros(*shape, device=DEV)
    assert decoding.cached_attention(z(0, 3, 2, 8), z(0, 3, 4, 2, 8), z(0, 3, 4, 2, 8)).shape == (0, 3, 2, 8)
    assert bool((decoding.cached_attention(z(2, 3, 2, 8) + 1, z(2, 3, 0, 2, 8), z(2, 3, 0, 2, 8)) == 0).all())
    assert [t.shape for t in decoding.beam_select(z(0, 3, 7), z(0, 3), 5)] == [(0, 5)] * 3
    decoding.reorder_states([], torch.zeros(2, 3, dtype=torch.int64, device=DEV))
    decoding.reorder_states([z(2, 3, 0, 4), z(2, 3, 4)], torch.zeros(2, 3, dtype=torch.int64, device=DEV))
    decoding.reorder_states([z(0, 3, 4)], torch.zeros(0, 3, dtype=torch.int64, device=DEV))


def test_calls_on_two_streams_at_once():
    from pam_b200 import decoding
    cases = [(_attention_case(8 + i), _select_case(8 + i)) for i in range(2)]
    want = [[decoding.cached_attention(**a), *decoding.beam_select(*b)] for a, b in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append([decoding.cached_attention(**cases[i][0]), *decoding.beam_select(*cases[i][1])])
    torch.cuda.synchronize()
    for mine, right in zip(got, want):
        for call in mine:
            for a, b in zip(call, right):
                assert torch.equal(a, b)


def test_calls_from_two_threads():
    """(kernels that need much shared memory, and different amounts of it, among them)"""
    from pam_b200 import decoding
    g = torch.Generator().manual_seed(40)
    randn = lambda *shape: torch.randn(*shape, generator=g).to(DEV)
    calls = []
    for i, (dim, beams) in enumerate(((256, 64), (128, 40))):
        a, b = _attention_case(18 + i), _select_case(18 + i)
        q, k, v, logits, scores = randn(2, 4, 2, dim) * 0.05, randn(2, 200 + i, 1, dim), randn(2, 200 + i, 1, dim), randn(2, beams, 600), randn(2, beams)
        calls.append(lambda a=a, b=b, q=q, k=k, v=v, logits=logits, scores=scores, beams=beams: [
            decoding.cached_attention(**a), *decoding.beam_select(*b), decoding.cached_attention(q, shared_k=k, shared_v=v),
            *decoding.beam_select(logits, scores, beams)])
    want = [call() for call in calls]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            try:
                for _ in range(100):
                    if not all(torch.equal(x, y) for x, y in zip(calls[i](), want[i])):
                        failures.append((i, "results"))
            except Exception as e:
                failures.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_a_step_captured_as_a_whole():
    """Attention with lengths on the device, selection, reordering: replayed as the lengths grow."""
    from pam_b200 import decoding
    g = torch.Generator().manual_seed(30)
    randn = lambda *shape: torch.randn(*shape, generator=g).to(DEV)
    own_k, own_v, q, table = randn(2, 3, 16, 2, 32), randn(2, 3, 16, 2, 32), randn(2, 3, 2, 32) * 0.2, randn(500, 64)
    start = [own_k.clone(), own_v.clone()]
    length, scores = torch.ones(2, 3, dtype=torch.int64, device=DEV), torch.zeros(2, 3, device=DEV)

    def step():
        out = decoding.cached_attention(q, own_k, own_v, length)
        best, beams, tokens = decoding.beam_select(out.flatten(2) @ table.t(), scores, 3)
        decoding.reorder_states([own_k, own_v], beams, length[:1, 0])
        return best, beams, tokens

    eager = []
    for n in (1, 5, 16):
        length.fill_(n)
        eager.append([*step(), own_k.clone(), own_v.clone()])
    for t, s in zip((own_k, own_v), start):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step()
    for t, s in zip((own_k, own_v), start):
        t.copy_(s)
    for n, want in zip((1, 5, 16), eager):
        length.fill_(n)
        graph.replay()
        for a, b in zip([*out, own_k, own_v], want):
            assert torch.equal(a, b)
