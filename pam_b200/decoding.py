"""Text generation on the GPU: attention over a key/value cache, the selection step of beam search, the reordering of
the states that belong to the beams, and sampling.

The reference's fairseq fork generates through the operators of its training graph: the whole chain of projections,
products and softmax per step (fairseq/modules/multihead_attention.py:618-783), log-probabilities sorted over beams
and vocabulary (fairseq/search.py:103-147) or drawn by sorted probabilities, states gathered by beam (fairseq/sequence_generator.py:380-388).  Here each of
the four is one call in the same PAM arithmetic, fp32 throughout.  None has a backward pass, and none takes an `offset`:
with one, the PAM softmax depends on the maximum of the whole tensor.
"""
import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib

MAX_HEAD_DIM = 256
MAX_BEAMS = 64
MAX_SELECTED = 64
MAX_SAMPLED = 1 << 18
_RANGE, _MAX_RANGES = 4092, 4096                # a beam's logits are worked on in ranges of so many; so many ranges may a group have


def _not_traced(what):
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be traced: its result would be recorded as a constant")


def _no_backward(what, *tensors):
    given = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given) or any(forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise RuntimeError(f"{what} has no derivative: call it under torch.no_grad() or on detached tensors")


def _fp32(name, t, dims):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
        raise TypeError(f"{name} must be an fp32 tensor, got {t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    return t


def _cache(name, k, v, lengths, lead, heads, dim):
    """Checks a pair of caches [*lead, slots, kv_heads, dim]; returns them with their lengths, cut where these are a number."""
    if (k is None) != (v is None):
        raise ValueError(f"{name} keys and values come together")
    if k is None:
        if lengths is not None:
            raise ValueError(f"{name} lengths without {name} keys and values")
        return None, None, None
    for what, t in ((f"{name} keys", k), (f"{name} values", v)):
        _fp32(what, t, len(lead) + 3)
        if tuple(t.shape[:len(lead)]) != lead or t.shape[-1] != dim:
            raise ValueError(f"{what} {tuple(t.shape)} do not go with queries of {lead} and head dimension {dim}")
        if dim > 1 and t.stride(-1) != 1:
            raise ValueError(f"{what}: the last dimension must be contiguous")
    if k.shape != v.shape:
        raise ValueError(f"{name} keys {tuple(k.shape)} and values {tuple(v.shape)} differ")
    if k.shape[-2] < 1 or heads % k.shape[-2]:
        raise ValueError(f"{heads} query heads cannot be shared out to {k.shape[-2]} key heads")
    slots = k.shape[-3]
    if isinstance(lengths, int) and not isinstance(lengths, bool):
        if not 0 <= lengths <= slots:
            raise ValueError(f"{name} length {lengths} outside the cache's {slots} slots")
        return k.narrow(-3, 0, lengths), v.narrow(-3, 0, lengths), None
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int64 or tuple(lengths.shape) != lead:
            raise ValueError(f"{name} lengths must be a number or an int64 tensor of shape {lead}")
        lengths = lengths.contiguous()
    return k, v, lengths


def cached_attention(q, own_k=None, own_v=None, own_lengths=None, *, shared_k=None, shared_v=None, shared_lengths=None):
    """PAM attention of single-token rows over cached keys and values: softmax(q k^T) v per head, as
    `fused.attention_heads` computes it for whole sequences (queries scaled by the caller).

    q           [groups, rows, heads, dim]: the new token of each row (beam, sample, sequence) of each group
    own_k/v     [groups, rows, slots, kv_heads, dim]: what each row has to itself (its own past), or None
    shared_k/v  [groups, positions, kv_heads, dim]: what the rows of a group have in common (the source sentence of its
                beams, a prompt), or None; read once for every eight rows times query heads of a key head
    lengths     how much of the cache is in use: a number, an int64 tensor ([groups, rows] own, [groups] shared), or None for
                all of it.  Lengths on the device are clamped to the slots; what lies beyond them is never read.

    kv_heads divides heads; key head i serves heads/kv_heads neighbouring query heads.  Caches may be any view whose last
    dimension is contiguous.  Returns [groups, rows, heads, dim]; a row that sees no position gets zeros.  The softmax
    shift is a whole number near the row's own maximum instead of the floor of the whole tensor's, which changes nothing
    but the rounding of the shifted scores.  Head dimensions up to 256, 2^20 rows times heads in a group, 2^30 positions, and groups x rows x heads x
    (2 + positions / 64) below 2^31."""
    if (host := _lib.host()) is not None:
        out = host.cached_attention(q, own_k, own_v, own_lengths, shared_k, shared_v, shared_lengths)
        if out is not None:
            return out
    _not_traced("cached_attention")
    _fp32("queries", q, 4)
    groups, rows, heads, dim = q.shape
    if own_k is None and shared_k is None:
        raise ValueError("cached_attention needs shared or own keys and values")
    if dim > MAX_HEAD_DIM:
        raise ValueError(f"head dimension {dim} is above {MAX_HEAD_DIM}")
    own_k, own_v, own_lengths = _cache("own", own_k, own_v, own_lengths, (groups, rows), heads, dim)
    shared_k, shared_v, shared_lengths = _cache("shared", shared_k, shared_v, shared_lengths, (groups,), heads, dim)
    if own_k is not None and shared_k is not None and own_k.shape[-2] != shared_k.shape[-2]:
        raise ValueError(f"shared keys have {shared_k.shape[-2]} heads, own keys {own_k.shape[-2]}")
    shared, own = (0 if t is None else t.shape[-3] for t in (shared_k, own_k))
    if rows * heads > 1 << 20 or shared + own > 1 << 30 or groups * rows * heads > (2 ** 31 - 1) // (2 + (shared + own) // 64):
        raise ValueError(f"{groups} groups of {rows} rows of {heads} heads over {shared + own} positions are too many for one call")
    _no_backward("cached_attention", q, own_k, own_v, shared_k, shared_v)
    dev = _lib.require_cuda(q, own_k, own_v, own_lengths, shared_k, shared_v, shared_lengths)
    if dim > 1 and q.stride(-1) != 1:
        q = q.contiguous()
    out = torch.empty(groups, rows, heads, dim, dtype=torch.float32, device=dev)
    if out.numel() == 0:
        return out
    kv_heads = (shared_k if own_k is None else own_k).shape[-2]
    strides = (ctypes.c_int64 * 17)(*q.stride()[:3], *(shared_k.stride()[:3] + shared_v.stride()[:3] if shared else (0,) * 6),
                                    *(own_k.stride()[:4] + own_v.stride()[:4] if own else (0,) * 8))
    ptr = lambda t, used=True: t.data_ptr() if t is not None and used else None
    handle = _lib.lib()
    sizes = (groups, rows, heads, kv_heads, dim, shared, own)
    ws_bytes = handle.pamk_cached_attention_workspace_bytes(*sizes)
    # (a buffer of this call alone: calls captured into different graphs share none)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    with _lib.device_guard(dev):
        status = handle.pamk_cached_attention(q.data_ptr(), out.data_ptr(), ptr(shared_k, shared), ptr(shared_v, shared), ptr(shared_lengths),
                                              ptr(own_k, own), ptr(own_v, own), ptr(own_lengths), *sizes, strides,
                                              ptr(ws), ws_bytes, _lib.stream_ptr(dev))
    _lib.check(status, "pamk_cached_attention")
    return out


def beam_select(logits, scores, k, banned=None):
    """One selection step of beam search: the k best continuations of every group over its beams and the vocabulary.

    logits  [groups, beams, vocabulary]: of the next token
    scores  [groups, beams]: the beams' scores so far; -inf (or NaN) for a beam that is not to be continued (at the first step all but
            one), whose logits are not read
    banned  bool, [vocabulary] or anything that broadcasts to the logits: tokens that must not be chosen (they keep their
            share of the probability)

    Returns (scores, beams, tokens), each [groups, k], best first: the new scores `scores + log_softmax(logits)` with the
    PAM log-softmax, the beam each continues (int64) and its token (int64).  Values are formed and compared in 64 bits; equal
    ones go to the lower beam, then to the larger logit, then to the lower token.  Logits of -1e30 or less, -inf among them, are masked: they have no
    share in the probability.  Masked and banned tokens and the tokens of beams that are not continued have score -inf and come
    last, also where a beam's logits hold NaN or overflow.  Up to 64 beams and k up to 64; beams times the vocabulary in ranges of 4092 tokens, the last
    one rounded up, up to 4096 (64 beams of 261888 tokens)."""
    if (host := _lib.host()) is not None:
        out = host.beam_select(logits, scores, k, banned)
        if out is not None:
            return out
    _not_traced("beam_select")
    _fp32("logits", logits, 3)
    _fp32("scores", scores, 2)
    groups, beams, vocab = logits.shape
    if tuple(scores.shape) != (groups, beams):
        raise ValueError(f"scores {tuple(scores.shape)} do not go with logits {tuple(logits.shape)}")
    if not isinstance(k, int) or isinstance(k, bool) or not 1 <= k <= min(MAX_SELECTED, beams * vocab):
        raise ValueError(f"k must be a number from 1 to {min(MAX_SELECTED, beams * vocab)}, got {k!r}")
    if beams > MAX_BEAMS:
        raise ValueError(f"{beams} beams are more than {MAX_BEAMS}")
    if beams * -(-vocab // _RANGE) > _MAX_RANGES:
        raise ValueError(f"{beams} beams of {vocab} tokens are more than {_MAX_RANGES} ranges of {_RANGE}")
    _no_backward("beam_select", logits, scores)
    dev = _lib.require_cuda(logits, scores, banned)
    if banned is not None:
        if not isinstance(banned, torch.Tensor) or banned.dtype != torch.bool:
            raise TypeError("banned must be a bool tensor")
        banned = banned.expand(groups, beams, vocab)
        if vocab > 1 and banned.stride(-1) != 1:
            banned = banned.contiguous()
    if vocab > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    best = torch.empty(groups, k, dtype=torch.float32, device=dev)
    which = torch.empty(2, groups, k, dtype=torch.int64, device=dev)
    if groups:
        handle = _lib.lib()
        ws_bytes = handle.pamk_beam_select_workspace_bytes(groups, beams, vocab, k)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with _lib.device_guard(dev):
            status = handle.pamk_beam_select(logits.data_ptr(), scores.data_ptr(), None if banned is None else banned.data_ptr(), best.data_ptr(),
                                             which[0].data_ptr(), which[1].data_ptr(), groups, beams, vocab, k, *logits.stride()[:2],
                                             *((0, 0) if banned is None else banned.stride()[:2]), ws.data_ptr(), ws_bytes,
                                             _lib.stream_ptr(dev))
        _lib.check(status, "pamk_beam_select")
    return best, which[0], which[1]


def _setting(name, value, shape, low, high, whole=False):
    """A number within [low, high], or a tensor of one for each row: (tensor or None, number)."""
    if isinstance(value, torch.Tensor):
        want = torch.int64 if whole else torch.float32
        if value.dtype != want or value.shape != shape:
            raise ValueError(f"{name} must be a number or a tensor {want} {tuple(shape)}, got {value.dtype} {tuple(value.shape)}")
        return value.contiguous(), 0
    if not isinstance(value, int if whole else (int, float)) or isinstance(value, bool) or not low <= value <= high:
        raise ValueError(f"{name} must be a {'whole ' if whole else ''}number from {low:g} to {high:g}, got {value!r}")
    return None, value


def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, banned=None):
    """Draws a token for every row of logits.

    logits   [..., vocabulary]: of the next token
    uniform  [...]: a number from [0, 1) for each row, in steps of 2^-24 as torch.rand gives them
    banned   bool, [vocabulary] or anything that broadcasts to the logits: tokens that must not be drawn (they keep their share of the probability)

    Tokens are drawn by the PAM softmax of pad(logits, temperature).  In the order of their probabilities, equal ones by number, there stay the first
    `top_k` (0: all), of these the ones before which less than `top_p` of their probability lies, of these the ones with at least `min_p` times the first one's.
    Each of the four is a number, or a tensor with one for each row (fp32, top_k int64; values out of range there are taken as the next one in range, a
    temperature that is not positive and finite leaves its row without a token).  The token is the first, by number, with which the probabilities that stay reach
    beyond `uniform`.  Probabilities are whole numbers of units of 2^-44 of the largest power of two, so that what is drawn depends on no rounding.

    Returns (tokens int64 [...], scores [...]): a score is the PAM log-softmax of pad(logits, temperature) at the token, over all tokens of the row.  Logits of -1e30 or less
    are masked.  A row that has no token to draw, or holds a NaN or a value beyond the PAM range, gets token -1 and score -inf.  Up to 262144 tokens."""
    if (host := _lib.host()) is not None:
        out = host.sample(logits, uniform, temperature, top_k, top_p, min_p, banned)
        if out is not None:
            return out
    _not_traced("sample")
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise ValueError("logits must be a tensor [..., vocabulary]")
    _fp32("logits", logits, logits.dim())
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    _fp32("uniform", uniform, len(lead))
    if uniform.shape != lead:
        raise ValueError(f"uniform {tuple(uniform.shape)} does not go with logits {tuple(logits.shape)}")
    if not 1 <= vocab <= MAX_SAMPLED:
        raise ValueError(f"a vocabulary of {vocab} is not from 1 to {MAX_SAMPLED}")
    temperature = _setting("temperature", temperature, lead, 2.0 ** -126, 2.0 ** 127)
    top_k = _setting("top_k", top_k, lead, 0, 2 ** 62, whole=True)
    top_p = _setting("top_p", top_p, lead, 2.0 ** -24, 1.0)
    min_p = _setting("min_p", min_p, lead, 0.0, 1.0)
    _no_backward("sample", logits, uniform)
    if banned is not None:
        if not isinstance(banned, torch.Tensor) or banned.dtype != torch.bool:
            raise TypeError("banned must be a bool tensor")
        # (one row of flags for all stays one)
        banned = banned.expand(vocab) if banned.dim() <= 1 else banned.expand(logits.shape).reshape(-1, vocab)
        banned = banned.contiguous()
    dev = _lib.require_cuda(logits, uniform, banned, *(s[0] for s in (temperature, top_k, top_p, min_p)))
    rows = uniform.numel()
    x = logits.reshape(rows, vocab)
    if vocab > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    uniform = uniform.contiguous()
    tokens = torch.empty(lead, dtype=torch.int64, device=dev)
    scores = torch.empty(lead, dtype=torch.float32, device=dev)
    ptr = lambda t: None if t is None else t.data_ptr()
    with _lib.device_guard(dev):
        status = _lib.lib().pamk_sample(x.data_ptr(), uniform.data_ptr(), ptr(banned), tokens.data_ptr(), scores.data_ptr(), rows, vocab, x.stride(0),
                                        vocab if banned is not None and banned.dim() == 2 else 0,
                                        *(v for t, n in (temperature, top_k, top_p, min_p) for v in (ptr(t), n)), _lib.stream_ptr(dev))
    _lib.check(status, "pamk_sample")
    return tokens, scores


def _span(t):
    """The bytes between a tensor's first and last element."""
    start = t.data_ptr()
    return start, start + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _rows_meet(apart, size, other, by_group, by_row, groups, rows):
    """Whether a row of `size` bytes of one state and a row of `other` bytes of another meet that lies `apart` bytes behind and has the same strides (two parts of
    one buffer, interleaved row by row, do not): whether apart + i by_group + j by_row is between -other and size for some differences i of groups and j
    of rows."""
    steps = sorted((step, n) for step, n in ((by_group, groups), (by_row, rows)) if n > 1)
    if steps and size <= apart <= steps[0][0] - other and (len(steps) == 1 or steps[1][0] >= steps[0][0] * steps[0][1]):
        return False                                      # (between two neighbouring rows, at the end of a group too: most often so)
    for j in range(1 - rows, rows):
        at = apart + j * by_row
        if groups == 1 or by_group == 0:
            i = 0
        else:
            i = max((-other - at) // by_group + 1, 1 - groups)                             # the first group that ends behind the row's start
        if i < groups and -other < at + i * by_group < size:
            return True
    return False


def _refuse_overlaps(states, moved, parents, used=None):
    """No two rows that move may share memory, neither of one tensor nor of two, and what says how they move may not lie in them."""
    spans = []
    for t, size in zip(states, moved):
        (groups, rows), (by_group, by_row) = t.shape[:2], (s * t.element_size() for s in t.stride()[:2])
        nested = ((groups == 1 or by_group >= (rows - 1) * by_row + size) and (rows == 1 or by_row >= size) or
                  (rows == 1 or by_row >= (groups - 1) * by_group + size) and (groups == 1 or by_group >= size))
        if not nested:
            raise ValueError(f"rows of a state of shape {tuple(t.shape)} and strides {t.stride()} overlap")
        spans.append((*_span(t), size, (by_group, by_row), (groups, rows)))
    spans.sort(key=lambda s: s[:2])
    read = [_span(t) for t in (parents, used) if t is not None]
    reach = []                                            # spans that may reach into the next one
    for s in spans:
        if any(s[0] < end and start < s[1] for start, end in read):
            raise ValueError("the parents, or the number of positions, lie in the memory of a state")
        reach = [r for r in reach if r[1] > s[0]]
        for r in reach:
            if r[3] != s[3] or _rows_meet(s[0] - r[0], r[2], s[2], *s[3], *s[4]):
                raise ValueError("two states share memory")
        reach.append(s)


def reorder_states(states, parents, used=None):
    """Moves the states of beams to where the beams go on, in place: state[g, r] = state[g, parents[g, r]] for every tensor
    [groups, beams, ...] in `states`, of any type.

    parents  int64 [groups, beams], the beam that each new beam continues; one outside the beams leaves its row as it is
    used     only the first `used` positions of the states' third dimension move (a number, or an int64 tensor of one element on the
             device); None: whole rows

    Each state's dimensions from the third on must be contiguous, and no two may share memory."""
    states = list(states)
    if (host := _lib.host()) is not None and host.reorder_states(states, parents, used):
        return
    _not_traced("reorder_states")
    if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int64 or parents.dim() != 2:
        raise ValueError("parents must be an int64 tensor [groups, beams]")
    groups, rows = parents.shape
    on_device = isinstance(used, torch.Tensor)
    if on_device:
        if used.dtype != torch.int64 or used.numel() != 1:
            raise ValueError("used must be a number or an int64 tensor of one element")
    elif used is not None and (not isinstance(used, int) or isinstance(used, bool) or used < 0):
        raise ValueError(f"used must be a number of positions, got {used!r}")
    if rows > MAX_BEAMS:
        raise ValueError(f"{rows} beams are more than {MAX_BEAMS}")
    moved, positions = [], []
    for t in states:
        if not isinstance(t, torch.Tensor) or t.dim() < 2 or tuple(t.shape[:2]) != (groups, rows):
            raise ValueError(f"every state must be a tensor [{groups}, {rows}, ...]")
        if used is not None and t.dim() < 3:
            raise ValueError("a state without positions cannot be moved in part")
        block = 1
        for n, s in reversed(list(zip(t.shape[2:], t.stride()[2:]))):
            if n > 1 and s != block:
                raise ValueError(f"a state of shape {tuple(t.shape)} and strides {t.stride()} is not contiguous within a row")
            block *= n
        slots = t.shape[2] if t.dim() > 2 else 1
        unit = block // slots * t.element_size() if slots else 0
        if used is not None and not on_device and used > slots:
            raise ValueError(f"{used} positions of a state with {slots}")
        positions.append(max(unit, 1))
        moved.append(unit * (slots if used is None or on_device else used))
    _no_backward("reorder_states", *states)
    if not states or parents.numel() == 0:
        return
    dev = _lib.require_cuda(*states, parents, used)
    parents = parents.contiguous()
    keep = [i for i, size in enumerate(moved) if size]
    states, moved, positions = ([x[i] for i in keep] for x in (states, moved, positions))
    if not states:
        return
    _refuse_overlaps(states, moved, parents, used if on_device else None)
    count = len(states)
    numbers = lambda values: (ctypes.c_int64 * count)(*values)
    with _lib.device_guard(dev):
        status = _lib.lib().pamk_reorder_states(
            (ctypes.c_void_p * count)(*[t.data_ptr() for t in states]), numbers(t.stride(0) * t.element_size() for t in states),
            numbers(t.stride(1) * t.element_size() for t in states), numbers(moved), numbers(positions), count, parents.data_ptr(),
            used.data_ptr() if on_device else None, groups, rows, _lib.stream_ptr(dev))
    _lib.check(status, "pamk_reorder_states")
    for t in states:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)
