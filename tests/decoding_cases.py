"""The operators of pam_b200.decoding from their definitions in 64 bits, on the CPU, with what their tests may be off by."""
import math

import torch

U = 2.0 ** -24                                   # half a step of fp32, relative
LOG2E = float(torch.tensor(math.log2(math.e), dtype=torch.float32))
INF = float("inf")


def _split(a):
    m, e = torch.frexp(a.abs())
    return torch.sign(a), 2 * m - 1, (e - 1).double()


def _rule(true, value):
    value = torch.where(true.abs() < 1e37, value, torch.nan)
    return torch.where(true.abs() < 1e-37, 0.0, value)


def pam(a, b):
    """Piecewise affine product of doubles."""
    a, b = torch.broadcast_tensors(torch.as_tensor(a, dtype=torch.float64), torch.as_tensor(b, dtype=torch.float64))
    (sa, fa, ea), (sb, fb, eb) = _split(a), _split(b)
    f = fa + fb
    carry = torch.floor(f)
    return _rule(a * b, torch.where((a == 0) | (b == 0), 0.0, sa * sb * torch.exp2(ea + eb + carry) * (1 + f - carry)))


def pad(a, b):
    a, b = torch.broadcast_tensors(torch.as_tensor(a, dtype=torch.float64), torch.as_tensor(b, dtype=torch.float64))
    (sa, fa, ea), (sb, fb, eb) = _split(a), _split(b)
    f = fa - fb
    carry = torch.floor(f)
    return _rule(a / b, torch.where(a == 0, 0.0, sa * sb * torch.exp2(ea - eb + carry) * (1 + f - carry)))


def exp2(x):
    whole = torch.floor(x)
    return torch.exp2(whole) * (1 + x - whole)


def attention(q, own_k, own_v, own_lengths, shared_k, shared_v, shared_lengths):
    """(out, bound): float64 [groups, rows, heads, dim] and what an fp32 evaluation may be off by.

    The bound, in units u = 2^-24, to first order: a score of `dim` products adds them with at most dim + 8 roundings, each of at most
    u times the sum A of their magnitudes; t = pam(s, log2 e) rises at most twice as fast as s.  t - m is rounded once (u |t - m|), so are
    the bracket of exp2 and its product, and e = exp2(t - m) changes relatively by no more than t does absolutely.  Half of what a score is off by
    reaches its own e and half the sum's: both are bounded by the largest of them, E.  The sum over n positions adds n u.  pad and pam
    follow their operands' relative changes at most twice as fast each.  The last sum adds n u of its terms' magnitudes W:
        |error| <= (4 (2 E + n u) + n u) W,    E = 2 (dim + 8) u A + u T + 2 u,    T = the largest |t - m| of a position with p > 0,
    and 2e-37 for each of the n terms, which may be flushed on one side and not on the other.
    """
    G, R, H, D = q.shape
    out, bound = torch.zeros(G, R, H, D, dtype=torch.float64), torch.zeros(G, R, H, D, dtype=torch.float64)
    for g in range(G):
        for r in range(R):
            keys, values = [], []
            for k, v, n, at in ((shared_k, shared_v, shared_lengths, (g,)), (own_k, own_v, own_lengths, (g, r))):
                if k is not None:
                    length = k.shape[-3] if n is None else n if isinstance(n, int) else int(n[at])
                    length = min(max(length, 0), k.shape[-3])
                    keys.append(k[at][:length])
                    values.append(v[at][:length])
            keys, values = (torch.cat(t).double().repeat_interleave(H // t[0].shape[1], 1) for t in (keys, values))      # [n, H, D]
            n = keys.shape[0]
            if n == 0:
                continue
            products = pam(q[g, r].double(), keys)
            s = products.sum(-1)                                                                                # [n, H]
            s = torch.where(s.abs() < 2.0 ** 128, s, torch.sign(s) * INF)                                       # (fp32 sums overflow)
            t = torch.where(s == -INF, -INF, pam(s, LOG2E))
            m = torch.floor(t.amax(0))
            e = torch.where(t == -INF, 0.0, exp2(t - m))
            p = pad(e, e.sum(0))
            terms = pam(p.unsqueeze(-1), values)
            out[g, r] = terms.sum(0)
            E = 2 * (D + 8) * U * products.abs().sum(-1).amax(0) + U * torch.where(p > 0, (t - m).abs(), 0.0).amax(0) + 2 * U
            bound[g, r] = (4 * (2 * E + n * U) + n * U).unsqueeze(-1) * terms.abs().sum(0) + 2e-37 * n
    return out, bound


def select(logits, scores, k, banned=None):
    """(scores, beams, tokens) by value, then lower beam, then larger logit, then lower token, one candidate after another."""
    G, R, V = logits.shape
    x = logits.double()
    ban = torch.zeros(G, R, V, dtype=torch.bool) if banned is None else banned.expand(G, R, V)
    best, beams, tokens = [], [], []
    for g in range(G):
        rows = []
        for r in range(R):
            masked = x[g, r] <= -1e30
            score = float(scores[g, r])
            # (terms as the kernels round them: 1 + fraction in fp32)
            t = torch.where(masked, -INF, pam(x[g, r], LOG2E)).float()
            top = torch.floor(t.max())
            whole = torch.floor(t)
            e = torch.where(masked, 0.0, (1 + (t - whole)).double() * torch.exp2((whole - top).double()))
            total = e.sum()
            finite = bool(total > 0) and bool(total < INF) and score > -INF
            if finite:
                mant, expo = torch.frexp(total)
                lse = float(pad(float(top) + float(expo) - 1 + (2 * float(mant) - 1), LOG2E))
                logit = torch.where(masked | ban[g, r], -INF, x[g, r])
                value = torch.where(logit == -INF, -INF, logit - lse + score)
            else:
                logit = value = torch.full((V,), -INF, dtype=torch.float64)
            order = torch.sort(logit, descending=True, stable=True).indices[:k]
            rows += [(-float(value[j]), r, i, int(j)) for i, j in enumerate(order)]
        rows.sort()
        best.append([-c[0] for c in rows[:k]])
        beams.append([c[1] for c in rows[:k]])
        tokens.append([c[3] for c in rows[:k]])
    return torch.tensor(best, dtype=torch.float64), torch.tensor(beams), torch.tensor(tokens)


def select_bound(values, exact_total=False):
    """What a selected score may be off by: its own rounding (u), and the logarithm's: each term of the sum is off by at most 1.5 u
    of itself, the affine log2 follows relative changes at most twice as fast and the division by log2 e no faster."""
    return U * values.abs() + 3 * U
