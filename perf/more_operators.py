"""The operators at the two ends of the vocabulary, as cases for timing and comparison.

Each case is a dict of plain values with a "kind":

  embed    pam.embedding: rows of a table by token, scaled in PAM arithmetic, with positions added and dropout; alone ("grad" is
           "none") or with the table's gradient, by products ("approx") or by slopes ("exact"), and that of learned positions
  dropout  pam.dropout: dropout from a counter-based generator, with or without a residual to add to; forward and backward
  sample   decoding.sample: a token for every row of logits from a given uniform number, with temperature, top-k, top-p and min-p

All data are fp32, the library's only type; tokens and seeds are int64.
"""
import math

import torch

own = False

DEV = "cuda"
LOG2E = 1.44269504088896340736


def listed():
    return [
        # a generation step: the last tokens of one sentence's five beams, all at one position
        dict(name="embed_step_1x5", kind="embed", rows=1, length=5, vocab=10000, dim=512, scaled=True, positions="one", pad=True, p=0.0, grad="none"),
        # the encoder's input in a training step of 128 sentences of up to 32 tokens
        dict(name="embed_train_128x32", kind="embed", rows=128, length=32, vocab=10000, dim=512, scaled=True, positions="table", pad=True, p=0.3, grad="approx"),
        # odd sizes, with the exact gradients and learned positions
        dict(name="embed_exact_9x333", kind="embed", rows=9, length=333, vocab=5003, dim=300, scaled=True, positions="learned", pad=False, p=0.1, grad="exact"),
        # long sequences over the vocabulary of a multilingual tokenizer
        dict(name="embed_train_32x1024", kind="embed", rows=32, length=1024, vocab=151643, dim=1024, scaled=True, positions="table", pad=True, p=0.1, grad="approx"),
        # the output of one sublayer for one sentence, added to what went in
        dict(name="dropout_32x512", kind="dropout", rows=32, width=512, p=0.3, residual=True, grad="approx"),
        # the same for a training batch of 128 sentences
        dict(name="dropout_4096x512", kind="dropout", rows=4096, width=512, p=0.3, residual=True, grad="approx"),
        # a large odd activation with the exact gradients
        dict(name="dropout_65537x1025", kind="dropout", rows=65537, width=1025, p=0.1, residual=False, grad="exact"),
        # one sentence's next token
        dict(name="sample_1x10000", kind="sample", rows=1, vocab=10000, temperature=1.0, top_k=50, top_p=0.95, min_p=0.0, banned=True, own_settings=False),
        # five samples of each of 128 sentences from the nucleus
        dict(name="sample_640x10000", kind="sample", rows=640, vocab=10000, temperature=0.9, top_k=0, top_p=0.9, min_p=0.0, banned=True, own_settings=False),
        # requests of a server, each with settings of its own
        dict(name="sample_64x50001_own", kind="sample", rows=64, vocab=50001, temperature=0.8, top_k=40, top_p=0.9, min_p=0.02, banned=False, own_settings=True),
        # the whole distribution over a large odd vocabulary
        dict(name="sample_256x151643", kind="sample", rows=256, vocab=151643, temperature=0.7, top_k=0, top_p=1.0, min_p=0.0, banned=False, own_settings=False),
        # the same from nuclei
        dict(name="sample_256x151643_nucleus", kind="sample", rows=256, vocab=151643, temperature=0.7, top_k=0, top_p=0.9, min_p=0.0, banned=False, own_settings=False),
    ]


def _spread(rng, lo, hi):
    """An integer between lo and hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("embed", "embed", "dropout", "sample", "sample"))
    if kind == "embed":
        tokens, vocab = _spread(rng, 1, 65536), _spread(rng, 100, 151643)
        dim = rng.choice((512, 512, 192, 64, 128, 256, 768, 1024, 4 * rng.randint(8, 256), rng.randint(16, 1024)))
        while tokens * dim > 33e6:
            tokens //= 2
        grad = rng.choice(("none", "approx", "approx", "exact"))
        length = min(tokens, _spread(rng, 1, 2048))
        return dict(kind=kind, rows=max(1, tokens // length), length=length, vocab=vocab, dim=dim, scaled=rng.random() < 0.8,
                    positions=rng.choice(("none", "one", "table", "table", "learned") if grad != "none" else ("none", "one", "table")),
                    pad=rng.random() < 0.6, p=rng.choice((0.0, 0.1, 0.3)), grad=grad)
    if kind == "dropout":
        width = rng.choice((512, 512, 192, 768, 1024, rng.randint(1, 2048)))
        return dict(kind=kind, rows=max(1, _spread(rng, 16, 67_000_000) // width), width=width, p=rng.choice((0.1, 0.1, 0.3, 0.5, round(rng.uniform(0.01, 0.9), 3))),
                    residual=rng.random() < 0.6, grad=rng.choice(("none", "approx", "approx", "exact")))
    vocab = _spread(rng, 30, 262144)
    return dict(kind=kind, rows=min(_spread(rng, 1, 1024), max(1, 38_000_000 // vocab)), vocab=vocab, temperature=round(rng.uniform(0.5, 1.5), 2),
                top_k=rng.choice((0, 0, 1, 10, 50, rng.randint(1, vocab))), top_p=rng.choice((1.0, 1.0, 0.5, 0.9, 0.95)),
                min_p=rng.choice((0.0, 0.0, 0.05, 0.2)), banned=rng.random() < 0.4, own_settings=rng.random() < 0.3)


# ---- inputs -----------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, s = case["kind"], dict(case)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEV)
    if kind != "sample":
        s["key"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), generator=g, device=DEV)      # what the mask is drawn from
    if kind == "embed":
        R, L, V, D = (case[k] for k in ("rows", "length", "vocab", "dim"))
        # words of a language: a few tokens are very frequent; sentences of different lengths, padded
        s["tokens"] = (torch.exp(rand(R, L) * math.log(V)).long() + 2).remainder(V)
        s["padding"] = 1 if case["pad"] else None
        if case["pad"]:
            ends = (L - rand(R, 1) * (L / 2)).ceil()
            s["tokens"].masked_fill_(torch.arange(L, device=DEV) >= ends, 1)
        s["weight"] = randn(V, D).mul_(D ** -0.5).requires_grad_(case["grad"] != "none")
        s["scale"] = math.sqrt(D) if case["scaled"] else None
        s["offsets"] = None if case["positions"] == "none" else randn(1 if case["positions"] == "one" else L, D).mul_(0.7)
        if case["positions"] == "learned":
            s["offsets"].requires_grad_()
        s["g"] = randn(R, L, D).mul_(1e-3) if case["grad"] != "none" else None
    elif kind == "dropout":
        shape = (case["rows"], case["width"])
        s["x"] = randn(*shape).requires_grad_(case["grad"] != "none")
        s["r"] = randn(*shape).requires_grad_(case["grad"] != "none") if case["residual"] else None
        s["g"] = randn(*shape).mul_(1e-3) if case["grad"] != "none" else None
    else:
        R, V = case["rows"], case["vocab"]
        s["logits"] = randn(R, V).mul_(2.5)
        # a few tokens of each row stand out, as they do in a trained model's
        at = (torch.randint(0, V, (R, 1), generator=g, device=DEV) + max(1, V // 20) * torch.arange(min(V, 20), device=DEV)) % V
        s["logits"].scatter_(1, at, randn(R, at.shape[1]).mul_(2.0).add_(8.0))
        s["uniform"] = rand(R)
        s["ban"] = None
        if case["banned"]:
            s["ban"] = torch.zeros(V, dtype=torch.bool, device=DEV)
            s["ban"][1] = True                                                                # the padding token
        if case["own_settings"]:
            s["temperature"] = case["temperature"] * (0.75 + 0.5 * rand(R))
            s["top_k"] = torch.where(rand(R) < 0.3, 0, torch.randint(1, 2 * max(case["top_k"], 10), (R,), generator=g, device=DEV))
            s["top_p"] = torch.where(rand(R) < 0.3, 1.0, 0.3 + 0.69 * rand(R))
            s["min_p"] = torch.where(rand(R) < 0.5, 0.0, 0.1 * rand(R))
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------

BIAS, FLUSH, PASS = 0x3F800000, 0x02081CEA, 0x7CF0BDC2     # bits of 1.0f, of the largest float below 1e-37, and below 1e37


def _ruled(true, candidate):
    """The range rule: nothing below 1e-37 in the true result, NaN from 1e37 on."""
    size = true.abs().view(torch.int32)
    out = torch.where(size <= PASS, candidate.view(torch.float32), torch.full((), float("nan"), device=true.device))
    return torch.where(size <= FLUSH, torch.zeros((), device=true.device), out)


def _number(v):
    return torch.full((), v, dtype=torch.float32, device=DEV)


def _pam(a, b):
    return _ruled(a * b, a.view(torch.int32) + b.view(torch.int32) - BIAS)


def _pad(a, b):
    return _ruled(a / b, a.view(torch.int32) - b.view(torch.int32) + BIAS)


def _slope(a, b):
    """d pam(a, b) / d a, a power of two with b's sign."""
    return (((a.view(torch.int32) & 0x7FFFFF) + b.view(torch.int32)) & -0x800000).view(torch.float32)


def _philox(key, count):
    """32 random bits for each of `count` elements (Philox4x32-10: Salmon, Moraes, Dror and Shaw 2011): the words of the blocks that
    the key's two halves make of the counters 0, 1, 2, ..."""
    low = 0xFFFFFFFF
    c0 = torch.arange((count + 3) // 4, device=DEV)
    c1, c2, c3 = (torch.zeros_like(c0) for _ in range(3))
    c1 += c0 >> 32
    c0 = c0 & low
    k0, k1 = key & low, (key >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).flatten()[:count]


def _kept(s, shape):
    """Which elements stay: those whose bits reach p 2^32, to the nearest whole number."""
    return (_philox(s["key"], math.prod(shape)) >= round(s["p"] * 2 ** 32)).view(shape)


def _keep_scale(p):
    return _number(1.0 / (1.0 - p))


def _through(g, y, s, kept):
    """What the gradient behind a dropout is before it, for its input y."""
    by = _keep_scale(s["p"])
    return torch.where(kept, _pam(g, by) if s["grad"] == "approx" else g * _slope(y, by), _number(0.0))


def _plain_embed(s):
    tokens, weight, pos = s["tokens"], s["weight"], s["offsets"]
    rows = weight[tokens]
    y = rows if s["scale"] is None else _pam(rows, _number(s["scale"]))
    if pos is not None:
        y = y + pos
    kept = _kept(s, y.shape) if s["p"] else None
    out = y if kept is None else torch.where(kept, _pam(y, _keep_scale(s["p"])), _number(0.0))
    if s["grad"] == "none":
        return out
    g = s["g"] if kept is None else _through(s["g"], y, s, kept)
    d_pos = g.sum(0, dtype=torch.float64).float() if s["positions"] == "learned" else None
    if s["scale"] is not None:
        by = _number(s["scale"])
        g = _pam(g, by) if s["grad"] == "approx" else g * _slope(rows, by)
    if s["padding"] is not None:
        g = torch.where((tokens == s["padding"]).unsqueeze(-1), _number(0.0), g)
    # (frequent tokens have thousands of terms)
    d_weight = torch.zeros(weight.shape, dtype=torch.float64, device=DEV).index_add_(0, tokens.flatten(), g.flatten(0, 1).double()).float()
    return [out, d_weight] + ([d_pos] if d_pos is not None else [])


def _plain_dropout(s):
    x, r = s["x"], s["r"]
    kept, by = _kept(s, x.shape), _keep_scale(s["p"])
    out = torch.where(kept, _pam(x, by), _number(0.0))
    if r is not None:
        out = out + r
    if s["grad"] == "none":
        return out
    return [out, _through(s["g"], x, s, kept)] + ([s["g"].clone()] if r is not None else [])


UNITS = 1 << 24


def _share(fraction, total):
    """Of whole numbers: floor(fraction total) for a fraction in steps of 2^-24."""
    part = torch.floor(fraction.double() * UNITS).long()
    return part * (total >> 24) + (part * (total & (UNITS - 1)) >> 24), part * (total & (UNITS - 1)) & (UNITS - 1)


def _share_up(fraction, total):
    whole, rest = _share(fraction, total)
    return whole + (rest > 0)


def _column(v, rows, dtype):
    return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), v, dtype=dtype, device=DEV)


def _plain_sample(s):
    x, ban = s["logits"], s["ban"]
    R, V = x.shape
    setting = lambda name, dtype: _column(s[name], R, dtype)
    x = _pad(x, setting("temperature", torch.float32))
    t = _pam(x, _number(LOG2E))
    # the exponential 2^whole (1 + f), f in steps of 2^-23, as a whole number of units of 2^-44 of the row's greatest power
    whole = torch.floor(t)
    mantissa = UNITS // 2 + torch.floor((t.double() - whole) * (UNITS // 2)).long()
    allowed = torch.ones_like(x, dtype=torch.bool) if ban is None else ~ban.expand(R, V)
    top = torch.where(allowed, whole, float("-inf")).amax(1, keepdim=True)
    below = (top - whole).clamp(max=100.0).long()
    weight = torch.where(allowed, torch.where(below <= 21, mantissa << (21 - below).clamp(min=0), mantissa >> (below - 21).clamp(0, 62)), 0)
    # in order of the exponentials, then of the tokens
    rank = torch.where(allowed, below * (UNITS // 2) - mantissa, 1 << 40)
    order = torch.sort(rank, dim=1, stable=True).indices
    ordered = weight.gather(1, order)
    place = torch.arange(V, device=DEV)
    top_k = setting("top_k", torch.int64)
    ordered = torch.where((top_k <= 0) | (place < top_k), ordered, 0)
    upto = ordered.cumsum(1)
    top_p = setting("top_p", torch.float32)
    bound = torch.where(top_p < 1.0, _share_up(top_p, upto[:, -1:]).clamp(min=1), upto[:, -1:])
    ordered = torch.where(upto - ordered < bound, ordered, 0)
    ordered = torch.where(ordered >= _share_up(setting("min_p", torch.float32), ordered[:, :1]), ordered, 0)
    weight = torch.zeros_like(weight).scatter_(1, order, ordered)
    upto = weight.cumsum(1)
    tokens = (upto <= _share(s["uniform"][:, None], upto[:, -1:])[0]).sum(1)
    # the logarithm of the probability among all tokens, in 64 bits
    shift = whole.amax(1, keepdim=True)
    terms = (1.0 + (t.double() - whole)) * torch.exp2((whole - shift).double())
    m, e = torch.frexp(terms.sum(1))
    log2 = shift[:, 0].double() + ((e - 1).double() + (2.0 * m - 1.0))
    by = _number(LOG2E).double()
    lse = (log2.view(torch.int64) - by.view(torch.int64) + torch.ones((), device=DEV, dtype=torch.float64).view(torch.int64)).view(torch.float64)
    lse = torch.where((log2 / by).abs() < 1e-37, 0.0, lse)
    return tokens, (x.gather(1, tokens[:, None])[:, 0].double() - lse).float()


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    kind = s["kind"]
    if not own:
        with torch.no_grad():
            return {"embed": _plain_embed, "dropout": _plain_dropout, "sample": _plain_sample}[kind](s)
    import pam_b200 as pam
    approx = s.get("grad") != "exact"
    if kind == "embed":
        out = pam.embedding(s["tokens"], s["weight"], s["scale"], s["offsets"], padding_idx=s["padding"], p=s["p"], seed=s["key"], approx_bwd=approx)
        leaves = [s["weight"]] + ([s["offsets"]] if s["positions"] == "learned" else [])
    elif kind == "dropout":
        out = pam.dropout(s["x"], s["p"], s["key"], residual=s["r"], approx_bwd=approx)
        leaves = [s["x"]] + ([s["r"]] if s["r"] is not None else [])
    else:
        from pam_b200 import decoding
        return decoding.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                               banned=s["ban"])
    if s["grad"] == "none":
        return out
    return [out.detach(), *torch.autograd.grad(out, leaves, s["g"])]


def work(case):
    if case["kind"] == "embed":
        N, V, D = case["rows"] * case["length"], case["vocab"], case["dim"]
        # (the distinct tokens of N that are drawn evenly over the logarithm)
        distinct = 1
        while distinct < min(N, V) and N / (distinct * math.log(V)) > 1.0:
            distinct += 1
        distinct = min(V, N, distinct + int(N * math.log(V / distinct) / math.log(V)))
        table = {"none": 0, "one": 1}.get(case["positions"], case["length"]) * D
        size, ops = 8 * N + 4 * (N * D + distinct * D + table), N * D * (case["scaled"] + (table > 0) + (case["p"] > 0))
        if case["grad"] != "none":
            size += 4 * (N * D + V * D) + 4 * table * (case["positions"] == "learned")
            ops += N * D * (1 + case["scaled"] + (case["p"] > 0))
        return {"bytes": size, "flops": ops}
    if case["kind"] == "dropout":
        n = case["rows"] * case["width"]
        r = case["residual"]
        forward = 4 * n * (2 + r)
        # (the residual's gradient is the incoming one; slopes take the input once more, which is one input all the same)
        backward = 0 if case["grad"] == "none" else 8 * n
        return {"bytes": forward + backward, "flops": n * (1 + r) + (n if case["grad"] != "none" else 0)}
    R, V = case["rows"], case["vocab"]
    return {"bytes": 4 * R * V + V * case["banned"] + 4 * R + 12 * R + 20 * R * case["own_settings"], "flops": 3 * R * V}


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


def _slope64(a, b):
    """The slope of a -> pam(a, b): 2^j, or 2^(j+1) where the fractions' sum reaches one."""
    _, fa, _ = _parts(a)
    sb, fb, eb = _parts(b)
    return sb * _pow2(eb + (fa + fb >= 1.0))


def _times(a, b):
    """The two 32-bit halves of the product of a 32-bit number and a constant, by 16 bits of the constant."""
    low, high = a * (b & 0xFFFF), a * (b >> 16)
    mid = high + (low >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _mask64(key, first, last, p):
    """Whether elements first .. last - 1 stay."""
    at = torch.arange(first, last, device=DEV)
    block, word = at // 4, at % 4
    c = [block % 2 ** 32, block // 2 ** 32, torch.zeros_like(at), torch.zeros_like(at)]
    key = int(key) % 2 ** 64
    for i in range(10):
        k = (key + i * 0x9E3779B9) % 2 ** 32, (key // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32
        (h0, l0), (h2, l2) = _times(c[0], 0xD2511F53), _times(c[2], 0xCD9E8D57)
        c = [h2 ^ c[1] ^ k[0], l2, h0 ^ c[3] ^ k[1], l0]
    return torch.stack(c).gather(0, word[None])[0] >= int(p * 2 ** 32 + 0.5)


def _exact_embed(s):
    tokens, D = s["tokens"], s["dim"]
    R, L = tokens.shape
    slopes = s["grad"] == "exact"
    by, keep = (_number(v).double() for v in (s["scale"] or 1.0, 1.0 / (1.0 - s["p"])))
    out = torch.empty(R, L, D, dtype=torch.float64, device=DEV)
    d_weight = torch.zeros(s["vocab"], D, dtype=torch.float64, device=DEV)
    d_pos = torch.zeros(L, D, dtype=torch.float64, device=DEV)
    some = max(1, (1 << 23) // (L * D))
    for r in range(0, R, some):
        ids = tokens[r:r + some]
        rows = s["weight"].detach()[ids].double()
        y = rows if s["scale"] is None else _pam64(rows, by)
        if s["offsets"] is not None:
            y = y + s["offsets"].detach().double()
        mask = _mask64(s["key"], r * L * D, (r + len(ids)) * L * D, s["p"]).view(-1, L, D) if s["p"] else None
        out[r:r + some] = y if mask is None else _pam64(y, keep) * mask
        if s["grad"] == "none":
            continue
        g = s["g"][r:r + some].double()
        if mask is not None:
            g = (g * _slope64(y, keep) if slopes else _pam64(g, keep)) * mask
        d_pos += g.sum(0)
        if s["scale"] is not None:
            g = g * _slope64(rows, by) if slopes else _pam64(g, by)
        live = torch.ones_like(ids, dtype=torch.bool) if s["padding"] is None else ids != s["padding"]
        d_weight.index_put_((ids[live],), g[live], accumulate=True)
    if s["grad"] == "none":
        return out
    return [out, d_weight] + ([d_pos] if s["positions"] == "learned" else [])


def _exact_dropout(s):
    x = s["x"].detach().double()
    keep = _number(1.0 / (1.0 - s["p"])).double()
    n = x.numel()
    mask = torch.cat([_mask64(s["key"], i, min(n, i + (1 << 23)), s["p"]) for i in range(0, n, 1 << 23)]).view(x.shape)
    out = _pam64(x, keep) * mask
    if s["r"] is not None:
        out += s["r"].detach().double()
    if s["grad"] == "none":
        return out
    g = s["g"].double()
    d = (g * _slope64(x, keep) if s["grad"] == "exact" else _pam64(g, keep)) * mask
    return [out, d] + ([g] if s["r"] is not None else [])


def _exact_sample(s):
    R, V = s["logits"].shape
    log2e = _number(LOG2E).double()
    tokens, scores = torch.empty(R, dtype=torch.int64, device=DEV), torch.empty(R, dtype=torch.float64, device=DEV)
    of = lambda name, r: s[name][r] if isinstance(s[name], torch.Tensor) else _number(s[name]) if isinstance(s[name], float) else s[name]
    for r in range(R):
        x = _pad64(s["logits"][r].double(), of("temperature", r).double())
        t = _pam64(x, log2e)
        live = torch.arange(V, device=DEV) if s["ban"] is None else (~s["ban"]).nonzero()[:, 0]
        # exponentials with 23 bits behind the point, in units of 2^-44 of the greatest power of two: whole numbers, exact in 64 bits
        _, fraction, exponent = _parts(_pow2(torch.floor(t)) * (1.0 + torch.floor((t - torch.floor(t)) * 2.0 ** 23) * 2.0 ** -23))
        exponent = exponent[live] - exponent[live].max()
        value = (1.0 + fraction[live]) * _pow2(exponent)
        by_value = torch.argsort(-value, stable=True)
        units = torch.floor(value * 2.0 ** 44).long()[by_value]
        k = int(of("top_k", r))
        if 0 < k < len(units):
            units, by_value = units[:k], by_value[:k]
        share = lambda name, total: -(-int(float(of(name, r)) * 2 ** 24) * int(total) // 2 ** 24)          # rounded up
        if float(of("top_p", r)) < 1.0:
            before = units.cumsum(0) - units
            n = int((before < max(share("top_p", units.sum()), 1)).sum())
            units, by_value = units[:n], by_value[:n]
        n = int((units >= share("min_p", units[0])).sum())
        units, by_value = units[:n], by_value[:n]
        in_order = torch.argsort(by_value)
        upto = units[in_order].cumsum(0)
        drawn = int(float(s["uniform"][r]) * 2 ** 24) * int(upto[-1]) // 2 ** 24
        tokens[r] = live[by_value[in_order[int((upto <= drawn).sum())]]]
        top = torch.floor(t.max())
        d = t - top
        _, fraction, exponent = _parts((_pow2(torch.floor(d)) * (1.0 + d - torch.floor(d))).sum())
        scores[r] = x[tokens[r]] - _pad64(top + exponent + fraction, log2e)
    return tokens, scores


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample" and case["rows"] > 400 and case["vocab"] > 100000:
        return None
    return {"embed": _exact_embed, "dropout": _exact_dropout, "sample": _exact_sample}[case["kind"]](s)
