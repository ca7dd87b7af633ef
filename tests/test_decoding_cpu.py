"""What the operators of pam_b200.decoding refuse, and their definitions against known values; no GPU needed."""
import ctypes

import pytest
import torch

import decoding_cases as oracle
from pam_b200 import _lib, decoding


def _attention(**change):
    case = dict(q=torch.zeros(2, 3, 4, 8), own_k=torch.zeros(2, 3, 5, 2, 8), own_v=torch.zeros(2, 3, 5, 2, 8),
                shared_k=torch.zeros(2, 6, 2, 8), shared_v=torch.zeros(2, 6, 2, 8))
    case.update(change)
    return decoding.cached_attention(**case)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 3, 32)), ValueError), (dict(q=torch.zeros(2, 3, 4, 8).half()), TypeError), (dict(q=None), TypeError),
    (dict(q=torch.zeros(2, 3, 3, 8)), ValueError), (dict(q=torch.zeros(2, 4, 4, 8)), ValueError), (dict(q=torch.zeros(2, 3, 4, 7)), ValueError),
    (dict(own_v=None), ValueError), (dict(shared_k=None), ValueError), (dict(own_v=torch.zeros(2, 3, 4, 2, 8)), ValueError),
    (dict(own_k=torch.zeros(2, 3, 5, 2, 8).double(), own_v=torch.zeros(2, 3, 5, 2, 8).double()), TypeError),
    (dict(shared_k=torch.zeros(2, 6, 1, 8), shared_v=torch.zeros(2, 6, 1, 8)), ValueError),
    (dict(shared_k=torch.zeros(2, 6, 0, 8), shared_v=torch.zeros(2, 6, 0, 8)), ValueError),
    (dict(shared_k=torch.zeros(2, 6, 8, 2).transpose(2, 3)), ValueError),
    (dict(own_lengths=6), ValueError), (dict(own_lengths=-1), ValueError), (dict(own_lengths=True), ValueError),
    (dict(own_lengths=torch.zeros(2, 3)), ValueError), (dict(own_lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(own_k=None, own_v=None, own_lengths=2), ValueError), (dict(own_k=None, own_v=None, shared_k=None, shared_v=None), ValueError),
    (dict(q=torch.zeros(2, 3, 4, 8, requires_grad=True)), RuntimeError), (dict(), RuntimeError),                     # (no GPU tensors)
])
def test_attention_refusals(change, error):
    with pytest.raises(error):
        _attention(**change)


def test_attention_refuses_wide_heads():
    with pytest.raises(ValueError, match="256"):
        decoding.cached_attention(torch.zeros(1, 1, 1, 257), torch.zeros(1, 1, 1, 1, 257), torch.zeros(1, 1, 1, 1, 257))


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(2, 30)), ValueError), (dict(logits=torch.zeros(2, 3, 10).half()), TypeError), (dict(scores=torch.zeros(3, 2)), ValueError),
    (dict(scores=torch.zeros(2, 3).double()), TypeError), (dict(k=0), ValueError), (dict(k=31), ValueError), (dict(k=True), ValueError),
    (dict(k=2.0), ValueError), (dict(logits=torch.zeros(2, 3, 100), k=65), ValueError),
    (dict(logits=torch.zeros(1, 65, 4), scores=torch.zeros(1, 65)), ValueError), (dict(logits=torch.zeros(2, 3, 10, requires_grad=True)), RuntimeError),
    (dict(), RuntimeError),
])
def test_select_refusals(change, error):
    case = dict(logits=torch.zeros(2, 3, 10), scores=torch.zeros(2, 3), k=4)
    case.update(change)
    with pytest.raises(error):
        decoding.beam_select(**case)


@pytest.mark.parametrize("states,parents,used,error", [
    ([torch.zeros(2, 3, 4)], torch.zeros(2, 3), None, ValueError), ([torch.zeros(2, 3, 4)], torch.zeros(6, dtype=torch.int64), None, ValueError),
    ([torch.zeros(3, 2, 4)], torch.zeros(2, 3, dtype=torch.int64), None, ValueError), ([torch.zeros(6, 4)], torch.zeros(2, 3, dtype=torch.int64), None, ValueError),
    ([torch.zeros(2, 3, 4)], torch.zeros(2, 3, dtype=torch.int64), 5, ValueError), ([torch.zeros(2, 3, 4)], torch.zeros(2, 3, dtype=torch.int64), -1, ValueError),
    ([torch.zeros(2, 3, 4)], torch.zeros(2, 3, dtype=torch.int64), 1.0, ValueError), ([torch.zeros(2, 3)], torch.zeros(2, 3, dtype=torch.int64), 1, ValueError),
    ([torch.zeros(2, 3, 4)], torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int64), ValueError),
    ([torch.zeros(2, 3, 5, 4).transpose(2, 3)], torch.zeros(2, 3, dtype=torch.int64), None, ValueError),
    ([torch.zeros(1, 65, 4)], torch.zeros(1, 65, dtype=torch.int64), None, ValueError),
    ([torch.zeros(2, 3, 4, requires_grad=True)], torch.zeros(2, 3, dtype=torch.int64), None, RuntimeError),
    ([torch.zeros(2, 3, 4)], torch.zeros(2, 3, dtype=torch.int64), None, RuntimeError),
])
def test_reorder_refusals(states, parents, used, error):
    with pytest.raises(error):
        decoding.reorder_states(states, parents, used)


def test_overlapping_states():
    parents = torch.zeros(2, 3, dtype=torch.int64)
    check = lambda *states: decoding._refuse_overlaps(list(states), [t[0, 0].numel() * t.element_size() for t in states], parents)
    buffer = torch.zeros(2, 3, 2, 8)
    check(buffer)
    check(buffer[:, :, 0], buffer[:, :, 1])                                        # interleaved
    check(buffer[:, :, 0, :4], buffer[:, :, 1], buffer[:, :, 0, 4:])
    check(torch.zeros(3, 2, 8).transpose(0, 1))
    check(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8))
    for states in ([buffer, buffer], [buffer[:, :, 0], buffer[:, :, 0]], [buffer, buffer[:, :, 1]], [buffer[:, :, 0], buffer[:, :, :, 4:].flatten(2)[:, :, :8], buffer[:, :, 0]],
                   [buffer[:, :, 0, :5], buffer[:, :, 0, 4:]], [torch.zeros(2, 1, 8).expand(2, 3, 8)], [torch.zeros(1, 3, 8).expand(2, 3, 8)],
                   [torch.zeros(100).as_strided((2, 3, 8), (24, 7, 1))], [torch.zeros(100).as_strided((2, 3, 8), (8, 8, 1))],
                   [parents.view(torch.float32).view(2, 3, 2)]):
        with pytest.raises(ValueError):
            check(*states)


def test_entry_points_check_their_arguments():
    h = _lib.lib()
    one = ctypes.addressof(ctypes.c_float(1.0))
    strides = (ctypes.c_int64 * 17)()
    call = lambda ptr, sizes, ws=None, n=0: h.pamk_cached_attention(ptr, ptr, ptr, ptr, None, None, None, None, *sizes, strides, ws, n, None)
    assert call(None, (1, 1, 1, 1, 4, 3, 0)) == -1 and call(one, (1, 1, 3, 2, 4, 3, 0)) == -1 and call(one, (1, 1, 1, 1, -4, 3, 0)) == -1
    assert call(one, (1, 1, 1, 1, 4, 3, 2)) == -1                                 # own positions without own keys
    assert call(one, (1, 1, 1, 1, 257, 3, 0)) == -2 and call(one, (1 << 30, 64, 1, 1, 4, 3, 0)) == -2
    assert call(one, (1, 1, 1, 1, 4, 3000, 0)) == -4 and call(one, (0, 1, 1, 1, 4, 3, 0)) == 0
    assert h.pamk_cached_attention_workspace_bytes(2, 3, 4, 2, 8, 6, 5) > 0 and h.pamk_cached_attention_workspace_bytes(2, 3, 4, 3, 8, 6, 5) == 0
    pick = lambda ptr, sizes, ws=None, n=0: h.pamk_beam_select(ptr, ptr, None, ptr, ptr, ptr, *sizes, 1, 1, 0, 0, ws, n, None)
    assert pick(None, (1, 1, 10, 2)) == -1 and pick(one, (1, 0, 10, 2)) == -1 and pick(one, (1, 65, 10, 2)) == -2 and pick(one, (1, 1, 10, 65)) == -2
    assert pick(one, (1, 1, 10, 11)) == -2 and pick(one, (1, 64, 1 << 30, 2)) == -2 and pick(one, (1, 1, 10, 2)) == -4 and pick(one, (0, 1, 10, 2)) == 0
    table = (ctypes.c_int64 * 1)(8)
    move = lambda states, count, parents, rows: h.pamk_reorder_states(states, table, table, table, table, count, parents, None, 1, rows, None)
    assert move(None, 1, one, 2) == -1 and move((ctypes.c_void_p * 1)(one), 1, None, 2) == -1 and move((ctypes.c_void_p * 1)(one), 1, one, 65) == -2
    assert move((ctypes.c_void_p * 1)(None), 1, one, 2) == -1 and move(None, 0, None, 2) == 0


def test_definitions(oracle=oracle):
    from oracle import build, pam_oracle
    build.build_oracle()
    g = torch.Generator().manual_seed(0)
    a, b = torch.randn(4000, generator=g), torch.randn(4000, generator=g)
    K = pam_oracle.kernels()
    assert torch.equal(oracle.pam(a, b).float(), K.pam_fwd(a, b, 1.0))
    assert torch.equal(oracle.pad(a, b).float(), K.pad_fwd(a, b, 1.0))
    # (x - floor(x) is off by half of u, one plus it by u)
    want = oracle.exp2(a.double())
    assert bool(((K.pa_exp_fwd(a, 2.0, 1.0).double() - want).abs() <= 1.5 * oracle.U * want).all())


def test_no_derivative_forward_either():
    from torch.autograd import forward_ad
    parents = torch.zeros(2, 3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: _attention(q=dual(torch.zeros(2, 3, 4, 8))), lambda: _attention(shared_v=dual(torch.zeros(2, 6, 2, 8))),
                     lambda: decoding.beam_select(torch.zeros(2, 3, 10), dual(torch.zeros(2, 3)), 4), lambda: decoding.reorder_states([dual(torch.zeros(2, 3, 4))], parents)):
            with pytest.raises(RuntimeError, match="derivative"):
                call()


def test_positions_in_a_state():
    states = [torch.zeros(2, 3, 4, dtype=torch.int64)]
    parents = torch.zeros(2, 3, dtype=torch.int64)
    decoding._refuse_overlaps(states, [32], parents, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="positions"):
        decoding._refuse_overlaps(states, [32], parents, states[0][1, 2, 3])


def test_positions_beyond_32_bits():
    h = _lib.lib()
    one = ctypes.addressof(ctypes.c_float(1.0))
    strides = (ctypes.c_int64 * 17)()
    for sizes in ((1, 1, 1, 1, 4, 1 << 30, 1 << 30), (1, 1, 1, 1, 4, 0, (1 << 30) + 1), (1, 1, 1, 1, 4, 1 << 40, 0)):
        assert h.pamk_cached_attention_workspace_bytes(*sizes) == 0
        assert h.pamk_cached_attention(one, one, one, one, None, one, one, None, *sizes, strides, None, 0, None) == -2
    assert h.pamk_cached_attention_workspace_bytes(1, 1, 1, 1, 4, 1 << 29, 1 << 29) > (1 << 30) * 4


def test_not_traced():
    k = torch.zeros(1, 1, 3, 1, 8)
    parents = torch.zeros(1, 2, dtype=torch.int64)
    for call, arg in ((lambda q: decoding.cached_attention(q, k, k), torch.zeros(1, 1, 1, 8)), (lambda x: decoding.beam_select(x, torch.zeros(1, 2), 2), torch.zeros(1, 2, 5)),
                      (lambda x: decoding.reorder_states([x], parents), torch.zeros(1, 2, 5))):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (arg,))
