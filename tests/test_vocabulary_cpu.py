"""Dropout, embedding and sampling without a GPU: the definitions that the GPU tests use, refusals, and the checks of the C entry points."""
import ctypes

import numpy as np
import pytest
import torch

import vocabulary_cases as define

import pam_b200 as pam
from pam_b200 import _lib, decoding


def test_random_bits():
    # (the generator's published answers)
    assert define.philox(0, 0) == (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    assert define.philox(2 ** 128 - 1, 2 ** 64 - 1) == (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)
    for seed, first, last, p in ((0, 0, 9, 0.5), (-5, 3, 30, 0.25), (2 ** 63 - 1, 2 ** 34 + 1, 2 ** 34 + 20, 0.9)):
        want = [define.philox(i // 4, seed % 2 ** 64)[i % 4] >= round(p * 2 ** 32) for i in range(first, last)]
        assert define.kept(seed, first, last, p).tolist() == want


def test_definitions_of_products():
    from oracle import build, pam_oracle
    build.build_oracle()
    K = pam_oracle.kernels()
    g = torch.Generator().manual_seed(0)
    x, d = torch.randn(1000, generator=g), torch.randn(1000, generator=g)
    assert torch.equal(define.pam(x, define.scale_of(0.3)).float(), K.pam_fwd(x, torch.full((1000,), define.scale_of(0.3)), 1.0))
    assert torch.equal((d.double() * define.slope(x.double(), define.scale_of(0.3))).float(), K.pam_bwd(x, torch.full((1000,), define.scale_of(0.3)), d, 1.0))


def test_definition_of_sampling():
    """Against the plain reading of it in floating point, away from ties and borders."""
    g = torch.Generator().manual_seed(1)
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.7, 0.0), (0, 1.0, 0.1), (9, 0.8, 0.02)):
        x = torch.randn(40, generator=g) * 2
        u = torch.rand((), generator=g)
        at = define.pad(x, define.F32(0.8))                                           # (a temperature is an fp32 number)
        t = define.pam(at, define.LOG2E)
        p = torch.exp2(torch.floor(t)) * (1 + t - torch.floor(t))
        p = p / p.sum()
        order = p.argsort(descending=True)
        stay = torch.zeros(40, dtype=torch.bool)
        stay[order[:top_k or 40]] = True
        q = torch.where(stay, p, 0.0)
        q = q / q.sum()
        cum = q[order].cumsum(0) - q[order]
        stay[order[cum >= top_p]] = False
        stay &= p >= min_p * p.max()
        q = torch.where(stay, p, 0.0)
        want = int((q.cumsum(0) <= u * q.sum()).sum())
        got, score, bound = define.sampled(x, u, 0.8, top_k, top_p, min_p, None)
        assert got == want and abs(score - float(at[got] - define.pad(torch.floor(t.max()) + _log2(t), define.LOG2E))) < 1e-9 and bound < 1e-6


def _log2(t):
    e = torch.exp2(torch.floor(t) - torch.floor(t.max())) * (1 + t - torch.floor(t))
    m, k = torch.frexp(e.sum())
    return k - 1 + 2 * m - 1


X = torch.zeros(4, 6)


@pytest.mark.parametrize("call, error", [
    (lambda: pam.dropout(X, 0.1), RuntimeError),                                     # a CPU tensor
    (lambda: pam.dropout(X.double(), 0.1), TypeError),
    (lambda: pam.dropout([1.0], 0.1), TypeError),
    (lambda: pam.dropout(X, 1.0), ValueError),
    (lambda: pam.dropout(X, -0.1), ValueError),
    (lambda: pam.dropout(X, float("nan")), ValueError),
    (lambda: pam.dropout(X, True), ValueError),
    (lambda: pam.dropout(X, torch.tensor(0.1)), ValueError),
    (lambda: pam.dropout(X, 0.1, residual=X[:3]), ValueError),
    (lambda: pam.dropout(X, 0.1, residual=X.half()), TypeError),
    (lambda: pam.dropout(X, 0.1, approx_bwd=(True, False)), ValueError),
    (lambda: pam.Dropout(1.0), ValueError),
    (lambda: pam.embedding(X.long(), X), RuntimeError),
    (lambda: pam.embedding(X, X), TypeError),
    (lambda: pam.embedding(X.long(), X.half()), TypeError),
    (lambda: pam.embedding(X.long(), X[0]), ValueError),
    (lambda: pam.embedding(X.long(), X, "2"), TypeError),
    (lambda: pam.embedding(X.long(), X, positions=X), ValueError),                   # tokens [4, 6]: positions are [6, 6]
    (lambda: pam.embedding(X.long(), X, positions=torch.zeros(6, 5)), ValueError),
    (lambda: pam.embedding(X.long(), X, positions=torch.zeros(0, 6)), ValueError),
    (lambda: pam.embedding(X.long(), X, padding_idx=4), ValueError),
    (lambda: pam.embedding(X.long(), X, p=1.0), ValueError),
    (lambda: pam.Embedding(4, 6, max_norm=1.0), ValueError),
    (lambda: pam.Embedding(4, 6, sparse=True), ValueError),
    (lambda: pam.Embedding(4, 6, p=2.0), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4)), RuntimeError),
    (lambda: decoding.sample(X.double(), torch.zeros(4)), TypeError),
    (lambda: decoding.sample(X, torch.zeros(3)), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4).double()), TypeError),
    (lambda: decoding.sample(torch.zeros(()), torch.zeros(())), ValueError),
    (lambda: decoding.sample(torch.zeros(2, 0), torch.zeros(2)), ValueError),
    (lambda: decoding.sample(torch.zeros(1, (1 << 18) + 1), torch.zeros(1)), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), temperature=0.0), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), temperature=float("inf")), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), temperature=torch.ones(3)), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), top_k=-1), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), top_k=2.0), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), top_k=torch.ones(4)), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), top_p=0.0), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), top_p=1.5), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), min_p=True), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), min_p=float("nan")), ValueError),
    (lambda: decoding.sample(X, torch.zeros(4), banned=torch.zeros(6)), TypeError),
    (lambda: decoding.sample(X, torch.zeros(4), banned=torch.zeros(5, dtype=torch.bool)), RuntimeError),
    (lambda: decoding.sample(X.clone().requires_grad_(), torch.zeros(4)), RuntimeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_seeds():
    from pam_b200.pam_ops import _seed
    cpu = torch.device("cpu")
    assert _seed(-3, cpu) == -3 and _seed(None, cpu).shape == (1,) and _seed(None, cpu).dtype == torch.int64
    for seed in (2 ** 63, True, 1.0, torch.zeros(2, dtype=torch.int64), torch.zeros(1)):
        with pytest.raises(ValueError):
            _seed(seed, cpu)


def test_without_dropout():
    x, r = torch.randn(3), torch.randn(3)
    assert pam.dropout(x, 0.0) is x and pam.dropout(x, 0.4, training=False) is x
    assert torch.equal(pam.dropout(x, 0.4, residual=r, training=False), r + x)
    assert pam.Dropout(0.4).eval()(x) is x


def test_modules():
    e = pam.Embedding(7, 4, padding_idx=-1, scale=2.0, p=0.1, approx_bwd=True)
    assert e.padding_idx == 6 and not e.weight[6].any() and e._get_name() == "pam.Embedding" and "scale=2.0" in repr(e) and list(e.state_dict()) == ["weight"]
    assert repr(pam.Dropout(0.25)) == "pam.Dropout(p=0.25, approx_bwd=False)"


def test_entry_points_check_their_arguments():
    h = _lib.lib()
    one = ctypes.addressof((ctypes.c_float * 64)())
    drop = lambda x, n, p: h.pamk_dropout(x, None, x, n, p, None, 0, 1.0, None)
    assert drop(None, 4, 0.5) == -1 and drop(one, -1, 0.5) == -1 and drop(one, 4, 0.0) == -1 and drop(one, 4, 1.0) == -1 and drop(one, 4, float("nan")) == -1
    assert drop(None, 0, 0.5) == 0 and h.pamk_dropout_bwd(one, None, one, 4, 0.5, None, 0, 1.0, None) == -1
    look = lambda tokens, table, pos, dy, out, sizes, p=0.0: h.pamk_embedding(tokens, table, pos, dy, out, *sizes, 1, 1.0, p, None, 0, 1.0, None)
    assert look(None, one, None, None, one, (2, 3, 4, 4, 0, 0)) == -1 and look(one, None, None, None, one, (2, 3, 4, 4, 0, 0)) == -1
    assert look(one, one, None, one, one, (2, 3, 4, 4, 0, 0)) == -1                  # a gradient of no dropout
    assert look(one, one, one, None, one, (3, 3, 4, 4, 4, 2)) == -1 and look(one, one, one, None, one, (2, 3, 4, 4, 4, 0)) == -1
    assert look(one, one, None, None, one, (2, (1 << 22) + 1, 4, 4, 0, 0)) == -2 and look(one, one, None, None, one, (1 << 31, 3, 4, 4, 0, 0)) == -2
    assert look(one, one, None, None, one, (2, 3, 4, 4, 0, 0), 1.0) == -1 and look(None, None, None, None, None, (0, 3, 4, 4, 0, 0)) == 0
    back = lambda tokens, dy, table, out, sizes, p=0.0, approx=1: h.pamk_embedding_bwd(tokens, dy, table, out, *sizes, -1, 1, 1.0, p, None, 0, 1.0, approx, None, 0, None)
    assert back(None, one, None, one, (2, 3, 4, 4)) == -1 and back(one, one, None, None, (2, 3, 4, 4)) == -1
    assert back(one, one, None, one, (2, 3, 4, 4), approx=0) == -1 and back(one, one, one, one, (2, 3, 4, 4), p=0.5, approx=0) == -1
    assert back(one, one, None, one, (2, 1 << 23, 4, 4)) == -2 and back(None, None, None, None, (0, 0, 4, 4)) == 0
    draw = lambda x, rows, vocab: h.pamk_sample(x, x, None, x, x, rows, vocab, vocab, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, None)
    assert draw(None, 1, 5) == -1 and draw(one, 1, 0) == -1 and draw(one, -1, 5) == -1 and draw(one, 1, (1 << 18) + 1) == -2 and draw(one, 1 << 28, 5) == -2
    assert draw(None, 0, 5) == 0
