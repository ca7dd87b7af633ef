"""The operators of text generation (pam_b200.decoding), as cases for timing and comparison.

Each case is a dict of plain values with a "kind":

  attention   decoding.cached_attention: single-token attention rows in PAM arithmetic.  `rows` rows (beams, samples) of each of
              `groups` groups attend to `shared` positions that the group has in common and to `own` positions of their own
  select      decoding.beam_select: the best `k` continuations over beams and vocabulary, from logits and running scores
  reorder     decoding.reorder_states: the rows of all cached states moved to the beams that go on, in place

All data are fp32, the library's only type; indices and lengths are int64.
"""
import math

import torch

own = False

DEV = "cuda"
LOG2E = 1.44269504088896340736


def listed():
    return [
        # cross-attention of one sentence's five beams over 32 source tokens, the 6+6 transformer's 4 heads of 128: all latency
        dict(name="attn_cross_1x5x32", kind="attention", groups=1, rows=5, heads=4, kv_heads=4, dim=128, shared=32, own=0, ragged=False),
        # self-attention of 128 sentences with five beams, 40 of 64 slots of each beam's cache in use
        dict(name="attn_self_128x5x64", kind="attention", groups=128, rows=5, heads=4, kv_heads=4, dim=128, shared=0, own=64, ragged=True),
        # cross-attention of that batch over padded sources of up to 48 tokens
        dict(name="attn_cross_128x5x48", kind="attention", groups=128, rows=5, heads=4, kv_heads=4, dim=128, shared=48, own=0, ragged=True),
        # eight continuations of each of four long documents, with up to 250 tokens of their own (heads of 64, as DeiT-tiny's)
        dict(name="attn_doc_4x8x8192", kind="attention", groups=4, rows=8, heads=16, kv_heads=16, dim=64, shared=8192, own=250, ragged=True),
        # one row over one very long context: few rows, the long axis split
        dict(name="attn_long_1x1x60001", kind="attention", groups=1, rows=1, heads=8, kv_heads=8, dim=64, shared=0, own=60001, ragged=False),
        # three samples of each of 16 prompts, four query heads on each key head
        dict(name="attn_grouped_16x3x2000", kind="attention", groups=16, rows=3, heads=32, kv_heads=8, dim=128, shared=2000, own=129, ragged=True),
        # the first step of one sentence: one beam alive, twice the beam asked for
        dict(name="select_first_1x5", kind="select", groups=1, rows=5, vocab=10000, k=10, first=True, banned="row"),
        # a step of 128 sentences with five beams over the 10000-word vocabulary
        dict(name="select_128x5x10000", kind="select", groups=128, rows=5, vocab=10000, k=10, first=False, banned="row"),
        # an odd vocabulary of a multilingual tokenizer, with tokens banned for each beam by itself
        dict(name="select_64x4x151643", kind="select", groups=64, rows=4, vocab=151643, k=8, first=False, banned="beam"),
        # the caches of one sentence: six layers' keys and values, 20 of 64 slots in use
        dict(name="reorder_1x5", kind="reorder", tensors=12, groups=1, rows=5, slots=64, used=20, width=512, moved=2),
        # the caches of 64 sentences
        dict(name="reorder_64x5", kind="reorder", tensors=12, groups=64, rows=5, slots=64, used=48, width=512, moved=2),
        # eight wide beams with long continuations
        dict(name="reorder_4x8", kind="reorder", tensors=12, groups=4, rows=8, slots=320, used=301, width=1024, moved=4),
    ]


def _spread(rng, lo, hi):
    """An integer between lo and hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "select", "select", "reorder"))
    if kind == "attention":
        dim = rng.choice((64, 64, 128, 128, 32, 256, 80, 96, 4 * rng.randint(1, 64), rng.randint(1, 256)))
        kv_heads, share = rng.choice(((1, 1), (2, 1), (3, 1), (4, 1), (8, 1), (16, 1), (1, 8), (2, 4), (4, 2), (8, 4))), rng.randint(0, 2)
        kv_heads, per = kv_heads
        groups, rows = _spread(rng, 1, 128), rng.choice((1, 1, 2, 3, 4, 5, 5, 8, rng.randint(1, 16)))
        shared = 0 if share == 0 else _spread(rng, 1, 65536)
        own_slots = 0 if share == 1 else _spread(rng, 1, 65536 if share == 0 and rows == 1 else 1024)
        # (no more than the largest listed case reads and computes)
        while (4 * groups * (shared + rows * own_slots) * kv_heads * dim * 2 > 150e6
               or groups * rows * per * kv_heads * dim * (shared + own_slots) * 2 > 500e6):
            groups, shared, own_slots = max(1, groups // 2), shared // 2 if groups == 1 else shared, own_slots // 2 if groups == 1 else own_slots
        return dict(kind=kind, groups=groups, rows=rows, heads=kv_heads * per, kv_heads=kv_heads, dim=dim, shared=shared,
                    own=own_slots if shared or own_slots else 1, ragged=rng.random() < 0.7)
    if kind == "select":
        rows, vocab = rng.choice((1, 2, 4, 5, 5, 8, rng.randint(1, 16))), _spread(rng, 100, 160000)
        groups = min(_spread(rng, 1, 256), max(1, 38_000_000 // (rows * vocab)))
        return dict(kind=kind, groups=groups, rows=rows, vocab=vocab, k=min(2 * rows, rows * vocab) if rng.random() < 0.8 else rng.randint(1, 32),
                    first=rng.random() < 0.2, banned=rng.choice(("none", "row", "beam")))
    rows = rng.choice((2, 3, 4, 5, 5, 8, rng.randint(2, 16)))
    slots, width = _spread(rng, 8, 512), 4 * rng.randint(16, 256)
    tensors = 2 * rng.randint(1, 12)
    groups = min(_spread(rng, 1, 128), max(1, 120_000_000 // (tensors * rows * slots * width)))
    return dict(kind=kind, tensors=tensors, groups=groups, rows=rows, slots=slots, used=rng.randint(1, slots), width=width,
                moved=rng.randint(1, rows - 1))


# ---- inputs -----------------------------------------------------------------------------------------------

def _lengths(case, count, slots):
    """Lengths spread from all of the slots down to half of them."""
    if not case["ragged"]:
        return [slots] * count
    return [slots - (i * (slots // 2)) // max(count - 1, 1) for i in range(count)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, s = case["kind"], dict(case)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
    G, R = case["groups"], case["rows"]
    if kind == "attention":
        H, K, D, P, S = case["heads"], case["kv_heads"], case["dim"], case["shared"], case["own"]
        # queries carry the factor 1/sqrt(dim) as the model's do; a few keys stand out, as they do in trained models
        s["q"] = randn(G, R, H, D).mul_(1.5 * D ** -0.5)
        spread = lambda n, count: torch.tensor(_lengths(case, n, count), device=DEV)[torch.randperm(n, generator=g, device=DEV)]
        for name, shape, slots in (("shared", (G, P, K, D), P), ("own", (G, R, S, K, D), S)):
            s[name + "_k"], s[name + "_v"] = (randn(*shape), randn(*shape)) if slots else (None, None)
            if slots:
                s[name + "_k"][..., :: 7, :, :] *= 1.7
        s["shared_lengths"] = spread(G, P) if P and case["ragged"] else None
        s["own_lengths"] = spread(G * R, S).view(G, R) if S and case["ragged"] else None
    elif kind == "select":
        V = case["vocab"]
        s["logits"] = randn(G, R, V).mul_(2.5)
        s["scores"] = randn(G, R).abs_().mul_(-3.0)
        if case["first"]:
            s["scores"] = torch.zeros(G, R, device=DEV)
            s["scores"][:, 1:] = float("-inf")
        s["banned_mask"] = None
        if case["banned"] == "row":
            s["banned_mask"] = torch.zeros(V, dtype=torch.bool, device=DEV)
            s["banned_mask"][1] = True                                                        # the padding token
        elif case["banned"] == "beam":
            s["banned_mask"] = torch.rand(G, R, V, generator=g, device=DEV) < 0.01
    else:
        s["states"] = [randn(G, R, case["slots"], case["width"]) for _ in range(case["tensors"])]
        # beams that go on stay where they are; the others take a copy of one of those
        order = torch.rand(G, R, generator=g, device=DEV).argsort(1)
        stay = R - case["moved"]
        s["parents"] = torch.arange(R, device=DEV).repeat(G, 1)
        moved = order[:, stay:]
        s["parents"].scatter_(1, moved, order[:, torch.arange(case["moved"], device=DEV) % stay])
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------

BIAS, FLUSH, PASS = 0x3F800000, 0x02081CEA, 0x7CF0BDC2     # bits of 1.0f, of the largest float below 1e-37, and below 1e37


def _ruled(true, candidate):
    """The range rule: nothing below 1e-37 in the true result, NaN from 1e37 on."""
    size = true.abs().view(torch.int32)
    out = torch.where(size <= PASS, candidate.view(torch.float32), torch.full((), float("nan"), device=true.device))
    return torch.where(size <= FLUSH, torch.zeros((), device=true.device), out)


def _pam(a, b):
    return _ruled(a * b, a.view(torch.int32) + b.view(torch.int32) - BIAS)


def _pad(a, b):
    return _ruled(a / b, a.view(torch.int32) - b.view(torch.int32) + BIAS)


def _power(e):
    """2^e for whole e, 0 below the normal numbers."""
    return torch.where(e < -126, 0, (e.clamp(-126, 127).int() + 127) << 23).int().view(torch.float32)


def _exp2(x):
    whole = torch.floor(x)
    return (1.0 + (x - whole)) * _power(whole)


def _live(lengths, slots, shape):
    """Which of the slots are in use, shaped to broadcast."""
    at = torch.arange(slots, device=DEV)
    return at < (torch.full((), slots, device=DEV) if lengths is None else lengths.unsqueeze(-1)).expand(*shape, 1)


def _rows_over(q, keys):
    """Scores [G, R, H, L] of rows q [G, R, H, D] on keys [G, R or 1, L, K, D], a row of each group at a time."""
    per = q.shape[2] // keys.shape[3]
    out = []
    for r in range(q.shape[1]):
        k = keys[:, min(r, keys.shape[1] - 1)].repeat_interleave(per, 2)                      # [G, L, H, D]
        out.append(_pam(q[:, r, None], k).sum(-1).transpose(1, 2))
    return torch.stack(out, 1)


def _weighted(p, values):
    """sum_j pam(p_j, v_j): p [G, R, H, L], values [G, R or 1, L, K, D]."""
    per = p.shape[2] // values.shape[3]
    out = []
    for r in range(p.shape[1]):
        v = values[:, min(r, values.shape[1] - 1)].repeat_interleave(per, 2)
        out.append(_pam(p[:, r].transpose(1, 2).unsqueeze(-1), v).sum(1))
    return torch.stack(out, 1)


def _plain_attention(s):
    q, (G, R) = s["q"], s["q"].shape[:2]
    scores, live, values = [], [], []
    if s["shared_k"] is not None:
        scores.append(_rows_over(q, s["shared_k"].unsqueeze(1)))
        live.append(_live(s["shared_lengths"], s["shared"], (G,))[:, None].expand(G, R, -1))
        values.append(s["shared_v"].unsqueeze(1))
    if s["own_k"] is not None:
        scores.append(_rows_over(q, s["own_k"]))
        live.append(_live(s["own_lengths"], s["own"], (G, R)))
        values.append(s["own_v"])
    t, live = torch.cat(scores, -1), torch.cat(live, -1).unsqueeze(2)
    t = torch.where(live, _pam(t, torch.full((), LOG2E, device=DEV)), torch.full((), float("-inf"), device=DEV))
    e = torch.where(live, _exp2(t - torch.floor(t.amax(-1, keepdim=True))), torch.zeros((), device=DEV))
    p = _pad(e, e.sum(-1, keepdim=True))
    p = torch.where(live, p, torch.zeros((), device=DEV))                                     # (a row without positions: zeros)
    parts = torch.split(p, [v.shape[2] for v in values], -1)
    return sum(_weighted(a, v) for a, v in zip(parts, values))


def _plain_select(s):
    x, scores, k = s["logits"], s["scores"], s["k"]
    G, R, V = x.shape
    t = _pam(x, torch.full((), LOG2E, device=DEV))
    whole = torch.floor(t)
    shift = whole.amax(-1, keepdim=True)
    # powers of two and a sum that lose nothing next to another beam's candidates take 64 bits
    total = ((1.0 + (t - whole)) * _power(whole - shift)).sum(-1, dtype=torch.float64)
    mantissa, exponent = torch.frexp(total)
    log2 = shift.squeeze(-1).double() + ((exponent - 1).double() + (2.0 * mantissa - 1.0))
    by = torch.full((), LOG2E, device=DEV).double()
    bias = torch.ones((), device=DEV, dtype=torch.float64).view(torch.int64)
    lse = (log2.view(torch.int64) - by.view(torch.int64) + bias).view(torch.float64)
    lse = torch.where((log2 / by).abs() < 1e-37, 0.0, lse)
    low = torch.full((), float("-inf"), device=DEV)
    x = torch.where((scores == float("-inf")).unsqueeze(-1), low, x)
    if s["banned_mask"] is not None:
        x = torch.where(s["banned_mask"], low, x)
    m = min(k, V)
    best, tokens = torch.sort(x, dim=-1, descending=True, stable=True)
    best, tokens = best[..., :m], tokens[..., :m]
    value = (best.double() - lse.unsqueeze(-1) + scores.double().unsqueeze(-1)).view(G, R * m)
    value, at = torch.sort(value, dim=-1, descending=True, stable=True)
    value, at = value[:, :k], at[:, :k]
    return value.float(), at // m, tokens.reshape(G, R * m).gather(1, at)


def _plain_reorder(s):
    for t in s["states"]:
        at = s["parents"][:, :, None, None].expand(-1, -1, s["used"], t.shape[-1])
        t[:, :, :s["used"]] = t[:, :, :s["used"]].gather(1, at)
    return s["states"]


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    kind = s["kind"]
    if own:
        from pam_b200 import decoding
        if kind == "attention":
            return decoding.cached_attention(s["q"], s["own_k"], s["own_v"], s["own_lengths"], shared_k=s["shared_k"],
                                             shared_v=s["shared_v"], shared_lengths=s["shared_lengths"])
        if kind == "select":
            return decoding.beam_select(s["logits"], s["scores"], s["k"], s["banned_mask"])
        decoding.reorder_states(s["states"], s["parents"], s["used"])
        return s["states"]
    with torch.no_grad():
        return {"attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder}[kind](s)


def work(case):
    G, R = case["groups"], case["rows"]
    if case["kind"] == "attention":
        H, K, D = case["heads"], case["kv_heads"], case["dim"]
        shared, mine = sum(_lengths(case, G, case["shared"])), sum(_lengths(case, G * R, case["own"]))
        lengths = 8 * (G * bool(case["shared"]) + G * R * bool(case["own"])) * case["ragged"]
        return {"bytes": 4 * (2 * G * R * H * D + 2 * K * D * (shared + mine)) + lengths,
                "flops": 4 * H * D * (R * shared + mine)}
    if case["kind"] == "select":
        V, beams = case["vocab"], G if case["first"] else G * R
        mask = {"none": 0, "row": V, "beam": beams * V}[case["banned"]]
        return {"bytes": 4 * beams * V + mask + 4 * G * R + 20 * G * case["k"], "flops": 3 * beams * V}
    moved = case["moved"]
    row = 4 * case["tensors"] * G * case["used"] * case["width"]
    return {"bytes": row * (moved + min(moved, R - moved)) + 8 * G * R, "flops": 0}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _parts(a):
    m, e = torch.frexp(a.abs())
    return torch.sign(a), 2.0 * m - 1.0, (e - 1).double()


def _pow2(e):
    return ((e.clamp(-1022, 1023).long() + 1023) << 52).view(torch.float64)


def _pam64(a, b):
    """2^i (1 + f) times 2^j (1 + g) = 2^(i+j) (1 + f + g), or 2^(i+j+1) (f + g) where f + g reaches one."""
    sa, fa, ea = _parts(a)
    sb, fb, eb = _parts(b)
    f = fa + fb
    return torch.where((a * b).abs() < 1e-37, 0.0, sa * sb * torch.where(f < 1.0, 1.0 + f, 2.0 * f) * _pow2(ea + eb))


def _pad64(a, b):
    sa, fa, ea = _parts(a)
    sb, fb, eb = _parts(b)
    f = fa - fb
    return torch.where((a / b).abs() < 1e-37, 0.0, sa * sb * torch.where(f >= 0.0, 1.0 + f, 1.0 + 0.5 * f) * _pow2(ea - eb))


def _exact_attention(s):
    q = s["q"].double()
    G, R, H, D = q.shape
    log2e = torch.full((), LOG2E, device=DEV).double()
    per = H // s["kv_heads"]
    out = torch.zeros(G, R, H, D, dtype=torch.float64, device=DEV)
    for g in range(G):
        n = s["shared"] if s["shared_lengths"] is None else int(s["shared_lengths"][g])
        for r in range(R):
            m = s["own"] if s["own_lengths"] is None else int(s["own_lengths"][g, r])
            keys, values = [], []
            if s["shared_k"] is not None:
                keys.append(s["shared_k"][g, :n])
                values.append(s["shared_v"][g, :n])
            if s["own_k"] is not None:
                keys.append(s["own_k"][g, r, :m])
                values.append(s["own_v"][g, r, :m])
            keys, values = (torch.cat(t).double().repeat_interleave(per, 1) for t in (keys, values))   # [L, H, D]
            if keys.shape[0] == 0:
                continue
            t = _pam64(_pam64(q[g, r], keys).sum(-1), log2e)                                  # [L, H]
            t = t - torch.floor(t.amax(0))
            e = _pow2(torch.floor(t)) * (1.0 + t - torch.floor(t))
            out[g, r] = _pam64(_pad64(e, e.sum(0)).unsqueeze(-1), values).sum(0)
    return out


def _exact_select(s):
    x, scores, k = s["logits"].double(), s["scores"].double(), s["k"]
    G, R, V = x.shape
    log2e = torch.full((), LOG2E, device=DEV).double()
    lse = torch.empty(G, R, dtype=torch.float64, device=DEV)
    for g in range(G):
        t = _pam64(x[g], log2e)
        top = torch.floor(t.amax(-1, keepdim=True))
        d = t - top
        total = (_pow2(torch.floor(d)) * (1.0 + d - torch.floor(d))).sum(-1)
        _, fraction, exponent = _parts(total)
        lse[g] = _pad64(top.squeeze(-1) + exponent + fraction, log2e)
    value = x - lse.unsqueeze(-1) + scores.unsqueeze(-1)
    value[scores == float("-inf")] = float("-inf")
    if s["banned_mask"] is not None:
        value = value.masked_fill(s["banned_mask"], float("-inf"))
    best, at = torch.sort(value.view(G, R * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    return best, at // V, at % V


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    if case["kind"] == "select":
        return _exact_select(s)
    index = torch.arange(case["groups"], device=DEV)[:, None]
    out = []
    for t in s["states"]:
        moved = t.clone()
        moved[:, :, :case["used"]] = t[index, s["parents"]][:, :, :case["used"]]
        out.append(moved)
    return out
