"""The two models of the reference's experiments as ``nn.Module``s built through the plugin API.

These are the module graphs of the reference's forks, reduced to what the PAM path touches, with
every swappable layer created the way the forks create it — from configuration strings through
``get_linear_factory / get_conv_factory / get_norm_factory / get_function_dict``
(shared/modules/factories.py:103-121, 124-199, 220-298):

* ``VisionTransformer``: DeiT-tiny of the timm fork (timm/models/vision_transformer.py:55-98,
  275-328, 437-440; timm/layers/mlp.py:25-38; timm/layers/patch_embed.py:36-47): patch embedding
  from the conv factory, qkv / proj / fc1 / fc2 / head from the linear factory, both attention
  products through the operator dictionary's ``bmm``.  On top of the fork's hooks the norm layers
  come from the norm factory and the attention scale and softmax from the operator dictionary
  (the configuration "PAM linear / LN / functional").
* ``Transformer``: the encoder-decoder of the fairseq fork at ``transformer_iwslt_de_en`` sizes
  (fairseq/modules/transformer_layer.py:38-84, 270-360; multihead_attention.py:96-149, 618-783;
  models/transformer/transformer_decoder.py:149-173, 455-463): projections and feed-forward layers
  from the linear factory, LayerNorms from the norm factory, query scaling, attention products,
  softmax and the embedding scale through the operator dictionary, decoder input and output
  embeddings tied so that the vocabulary projection is a layer of the linear factory too, and the
  label-smoothed loss of criterions/label_smoothed_cross_entropy.py:36-54 through the loss
  operator dictionary.

Parameter names follow the forks (``blocks.3.attn.qkv.weight``, ``encoder.layers.0.self_attn.
q_proj.weight`` ...), so state dictionaries interchange with models built from the stock layers.
``load_parameters`` fills a model from the flat dictionaries of ``pam_b200.steps`` (the functional
form of the same graphs), which is how the tests check that both forms agree bit for bit.
"""
import math

import torch
import torch.nn.functional as F
from torch import nn

from . import decoding, factories, fused
from .pam_opt import _pam_binding
from .steps import DeitConfig, TransformerConfig, sinusoidal_positions


# ---- DeiT-tiny (timm fork) -----------------------------------------------------------------------------

class Attention(nn.Module):
    def __init__(self, dim, num_heads, qkv_bias, linear_factory, ops):
        super().__init__()
        self.num_heads, self.scale, self.ops = num_heads, (dim // num_heads) ** -0.5, ops
        self.qkv = linear_factory(dim, dim * 3, bias=qkv_bias)
        self.proj = linear_factory(dim, dim)

    def forward(self, x):
        B, N, C = x.shape
        qkv = self.qkv(x)
        bound = _pam_binding(self.ops, ("bmm", "softmax", "mul"))
        if bound is not None and fused.attention_supported(qkv, self.num_heads, bound.get("approx_bwd", False)):
            # the same products, scaling and softmax on strided views of qkv: no copies around them
            return self.proj(fused.attention_qkv(qkv, self.num_heads, self.scale, offset=bound.get("offset")))
        qkv = qkv.reshape(B, N, 3, self.num_heads, C // self.num_heads).permute(2, 0, 3, 1, 4)
        q, k, v = qkv.unbind(0)
        attn = self.ops["bmm"](q.flatten(0, 1), k.transpose(-2, -1).flatten(0, 1))
        attn = self.ops["softmax"](self.ops["mul"](attn, self.scale), dim=-1)
        x = self.ops["bmm"](attn, v.flatten(0, 1)).view(B, self.num_heads, N, C // self.num_heads)
        return self.proj(x.transpose(1, 2).reshape(B, N, C))


class Mlp(nn.Module):
    def __init__(self, in_features, hidden_features, linear_factory):
        super().__init__()
        self.fc1 = linear_factory(in_features, hidden_features, bias=True)
        self.act = nn.GELU()
        self.fc2 = linear_factory(hidden_features, in_features, bias=True)

    def forward(self, x):
        return self.fc2(self.act(self.fc1(x)))


class Block(nn.Module):
    def __init__(self, dim, num_heads, hidden, norm_layer, linear_factory, ops):
        super().__init__()
        self.norm1 = norm_layer(dim)
        self.attn = Attention(dim, num_heads, True, linear_factory, ops)
        self.norm2 = norm_layer(dim)
        self.mlp = Mlp(dim, hidden, linear_factory)

    def forward(self, x):
        x = x + self.attn(self.norm1(x))
        return x + self.mlp(self.norm2(x))


class PatchEmbed(nn.Module):
    def __init__(self, patch, channels, dim, conv_factory):
        super().__init__()
        self.proj = conv_factory(channels, dim, kernel_size=patch, stride=patch)

    def forward(self, x):
        return self.proj(x).flatten(2).transpose(1, 2)


class VisionTransformer(nn.Module):
    def __init__(self, cfg=DeitConfig(), linear_cfg="standard", conv_cfg="standard", norm_cfg="layer_norm",
                 functional_cfg="torch"):
        super().__init__()
        self.cfg = cfg
        linear_factory = factories.get_linear_factory(linear_cfg)
        norm_factory = factories.get_norm_factory(norm_cfg)
        norm_layer = lambda dim: norm_factory(dim, eps=cfg.eps)
        ops = factories.get_function_dict(functional_cfg)
        self.patch_embed = PatchEmbed(cfg.patch, cfg.channels, cfg.dim, factories.get_conv_factory(conv_cfg))
        self.cls_token = nn.Parameter(torch.zeros(1, 1, cfg.dim))
        self.pos_embed = nn.Parameter(torch.zeros(1, cfg.tokens, cfg.dim))
        self.blocks = nn.Sequential(*[Block(cfg.dim, cfg.heads, cfg.mlp, norm_layer, linear_factory, ops)
                                      for _ in range(cfg.depth)])
        self.norm = norm_layer(cfg.dim)
        self.head = linear_factory(cfg.dim, cfg.classes)

    def forward(self, images):
        x = self.patch_embed(images)
        x = torch.cat([self.cls_token.expand(x.shape[0], -1, -1), x], dim=1) + self.pos_embed
        x = self.norm(self.blocks(x))
        return self.head(x[:, 0])

    def load_parameters(self, p):
        """Fills the model from the flat dictionary of `steps.deit_params`."""
        names = {"ln1": "norm1", "qkv": "attn.qkv", "proj": "attn.proj", "ln2": "norm2", "fc1": "mlp.fc1", "fc2": "mlp.fc2"}
        state = {"patch_embed.proj.weight": p["patch.w"], "patch_embed.proj.bias": p["patch.b"], "cls_token": p["cls"],
                 "pos_embed": p["pos"], "norm.weight": p["norm.w"], "norm.bias": p["norm.b"],
                 "head.weight": p["head.w"], "head.bias": p["head.b"]}
        for key, value in p.items():
            if key.startswith("blocks."):
                _, index, rest = key.split(".", 2)
                stem, kind = rest.split(".")
                state[f"blocks.{index}.{names[stem]}.{'weight' if kind == 'w' else 'bias'}"] = value
        self.load_state_dict({k: v.detach() for k, v in state.items()})
        return self


# ---- encoder-decoder transformer (fairseq fork) ----------------------------------------------------------

class MultiheadAttention(nn.Module):
    """The explicit (non-fused) branch the fork takes when custom operators are configured."""

    def __init__(self, embed_dim, num_heads, linear_factory, op_dict):
        super().__init__()
        self.num_heads, self.head_dim = num_heads, embed_dim // num_heads
        self.scaling = self.head_dim ** -0.5
        self.k_proj = linear_factory(embed_dim, embed_dim, bias=True)
        self.v_proj = linear_factory(embed_dim, embed_dim, bias=True)
        self.q_proj = linear_factory(embed_dim, embed_dim, bias=True)
        self.out_proj = linear_factory(embed_dim, embed_dim, bias=True)
        self.gain_op, self.bmm_op, self.softmax_op = op_dict["mul"], op_dict["bmm"], op_dict["softmax"]
        self.ops = op_dict

    def forward(self, query, memory, attn_mask=None):
        B, T, d = query.shape
        S, H, hd = memory.shape[1], self.num_heads, self.head_dim
        q = self.gain_op(self.q_proj(query), self.scaling)
        k, v = self.k_proj(memory), self.v_proj(memory)
        bound = _pam_binding(self.ops, ("bmm", "softmax"))
        if bound is not None and fused.attention_heads_supported(q, k, v, H, attn_mask, bound.get("approx_bwd", False)):
            # the same products, mask and softmax on strided views of the projections: no copies around them
            return self.out_proj(fused.attention_heads(q, k, v, H, attn_mask, offset=bound.get("offset")))
        split = lambda t, L: t.reshape(B, L, H, hd).transpose(1, 2).reshape(B * H, L, hd)
        w = self.bmm_op(split(q, T), split(k, S).transpose(1, 2))
        if attn_mask is not None:
            w = w + attn_mask
        w = self.softmax_op(w, dim=-1)
        ctx = self.bmm_op(w, split(v, S)).reshape(B, H, T, hd).transpose(1, 2).reshape(B, T, d)
        return self.out_proj(ctx)

    def cache(self, memory):
        """The keys and values of `memory` [..., length, dim], heads apart: [..., length, heads, head_dim]."""
        return tuple(f(memory).unflatten(-1, (self.num_heads, self.head_dim)) for f in (self.k_proj, self.v_proj))

    def step(self, query, own=None, own_length=None, shared=None, shared_lengths=None):
        """One new token of each row, [groups, rows, dim], over cached keys and values: each row's `own` ones, of which `own_length`
        positions are in use, or those that the rows of a group have in common (`shared`, `shared_lengths` of them)."""
        q = self.gain_op(self.q_proj(query), self.scaling).unflatten(-1, (self.num_heads, self.head_dim))
        bound = _pam_binding(self.ops, ("bmm", "softmax"))
        if _plain(bound, q) and self.head_dim <= decoding.MAX_HEAD_DIM:
            kv = dict(zip(("own_k", "own_v"), own)) if shared is None else dict(zip(("shared_k", "shared_v"), shared))
            ctx = decoding.cached_attention(q, own_lengths=own_length, shared_lengths=shared_lengths, **kv)
            return self.out_proj(ctx.flatten(2))
        G, R, H, hd = q.shape
        if shared is None:                                       # rows and heads apart, one query each
            q, k, v = q.reshape(G * R * H, 1, hd), *(t[:, :, :own_length].transpose(2, 3).reshape(G * R * H, -1, hd) for t in own)
        else:                                                    # heads apart, a group's rows together
            q, k, v = q.transpose(1, 2).reshape(G * H, R, hd), *(t.transpose(1, 2).reshape(G * H, -1, hd) for t in shared)
        w = self.bmm_op(q, k.transpose(1, 2))
        if shared_lengths is not None:
            w = w + _beyond(shared_lengths, k.shape[1]).repeat_interleave(H, 0)
        ctx = self.bmm_op(self.softmax_op(w, dim=-1), v)
        ctx = ctx.view(G, R, H, hd) if shared is None else ctx.view(G, H, R, hd).transpose(1, 2)
        return self.out_proj(ctx.reshape(G, R, H * hd))


def _plain(bound, t):
    """Whether the operators of `decoding` stand for the dictionary's on this tensor: PAM functions without an offset, fp32 on a GPU."""
    return bound is not None and bound.get("offset") in (None, 1.0) and t.is_cuda and t.dtype == torch.float32


def _beyond(lengths, slots):
    """-inf at the positions from each length on, 0 before: [count, 1, slots]."""
    beyond = torch.arange(slots, device=lengths.device) >= lengths[:, None]
    return torch.zeros(beyond.shape, device=lengths.device).masked_fill_(beyond, float("-inf")).unsqueeze(1)


class TransformerLayer(nn.Module):
    """Post-norm encoder layer, or decoder layer when `cross` is set (transformer_layer.py)."""

    def __init__(self, cfg, cross, linear_factory, norm_layer, op_dict):
        super().__init__()
        self.self_attn = MultiheadAttention(cfg.dim, cfg.heads, linear_factory, op_dict)
        self.self_attn_layer_norm = norm_layer(cfg.dim)
        if cross:
            self.encoder_attn = MultiheadAttention(cfg.dim, cfg.heads, linear_factory, op_dict)
            self.encoder_attn_layer_norm = norm_layer(cfg.dim)
        self.fc1 = linear_factory(cfg.dim, cfg.ffn)
        self.fc2 = linear_factory(cfg.ffn, cfg.dim)
        self.final_layer_norm = norm_layer(cfg.dim)
        self.cross = cross

    def forward(self, x, memory=None, self_mask=None):
        x = self.self_attn_layer_norm(x + self.self_attn(x, x, self_mask))
        if self.cross:
            x = self.encoder_attn_layer_norm(x + self.encoder_attn(x, memory))
        return self.final_layer_norm(x + self.fc2(torch.relu(self.fc1(x))))

    def step(self, x, own, position, shared, shared_lengths):
        """The decoder layer on one new token of each row, [groups, rows, dim]: its key and value go to `position` of the row's own
        cache, the source's are those of its group."""
        for cache, new in zip(own, self.self_attn.cache(x)):
            cache[:, :, position] = new
        x = self.self_attn_layer_norm(x + self.self_attn.step(x, own=own, own_length=position + 1))
        x = self.encoder_attn_layer_norm(x + self.encoder_attn.step(x, shared=shared, shared_lengths=shared_lengths))
        return self.final_layer_norm(x + self.fc2(torch.relu(self.fc1(x))))


def _ordinary_call(device):
    """Whether a tensor made now may be kept: not one that belongs to a trace, a transform, a dispatch mode or a compiler,
    nor one that a captured graph would go on reading after it was replaced."""
    return not (torch.jit.is_tracing() or torch.compiler.is_compiling() or torch._C._are_functorch_transforms_active()
                or torch._C._len_torch_dispatch_stack() or (device.type == "cuda" and torch.cuda.is_current_stream_capturing()))


def _kept(module, name, length, device, make, cut):
    """A constant table for sequences of `length`: `cut` of the one that `module` keeps, on each device, for the longest
    sequence so far (to the next power of two), made by `make`."""
    if not _ordinary_call(device):
        return cut(make(length, device), length)
    tables = module.__dict__.setdefault("_kept_tables", {})
    stream = torch._C._cuda_getCurrentRawStream(device.index) if device.type == "cuda" else None
    entry = tables.get((name, device))                       # (stream that made it, table, last length, its cut)
    if entry is None or entry[1].device != device:
        entry = (stream, None, 0, None)
    owner, table, last, view = entry
    if table is not None and stream != owner:
        table.record_stream(torch.cuda.current_stream(device))    # (a longer one may replace it while the stream still reads it)
    if last != length:
        with torch.inference_mode(False):
            if table is None or table.shape[0] < length:
                owner, table = stream, make(1 << (length - 1).bit_length(), device)
                if stream is not None:
                    torch.cuda.current_stream(device).synchronize()      # (other streams use it without waiting for this one)
            view = cut(table, length)
        tables[name, device] = (owner, table, length, view)
    return view


class _Stack(nn.Module):
    def __init__(self, cfg, layers, cross, linear_factory, norm_layer, op_dict):
        super().__init__()
        self.cfg, self.op_dict = cfg, op_dict
        self.embed_tokens = nn.Embedding(cfg.vocab, cfg.dim, padding_idx=cfg.pad)
        self.embed_scale = math.sqrt(cfg.dim)
        self.layers = nn.ModuleList([TransformerLayer(cfg, cross, linear_factory, norm_layer, op_dict) for _ in range(layers)])

    def _positions(self, length, device):
        """The first rows of the sinusoidal table, which take the host and a copy that waits to make."""
        return _kept(self, "positions", length, device, lambda n, d: sinusoidal_positions(n, self.cfg.dim, self.cfg.pad, d),
                     lambda table, n: table[:n])

    def _future(self, length, device):
        """-inf above the diagonal."""
        return _kept(self, "future", length, device, lambda n, d: torch.full((n, n), float("-inf"), device=d).triu(1),
                     lambda table, n: table[:n, :n])

    def embed(self, tokens):
        x = self.op_dict["mul"](self.embed_scale, self.embed_tokens(tokens))
        return x + self._positions(tokens.shape[1], tokens.device)


def _select(ops, logits, scores, count, banned):
    """The `count` best continuations: (scores, beams, tokens) as `decoding.beam_select` gives them."""
    bound = _pam_binding(ops, ("log_softmax",))
    if _plain(bound, logits):
        return decoding.beam_select(logits, scores, count, banned)
    values = ops["log_softmax"](logits, dim=-1) + scores.unsqueeze(-1)
    values, at = values.masked_fill(banned, float("-inf")).flatten(1).topk(count, 1)
    return values, at // logits.shape[-1], at % logits.shape[-1]


def _reorder(states, parents, used):
    if parents.is_cuda:
        return decoding.reorder_states(states, parents, used)
    group = torch.arange(parents.shape[0])[:, None]
    for t in states:
        t[:, :, :used] = t[group, parents, :used]


class Transformer(nn.Module):
    def __init__(self, cfg=TransformerConfig(), linear_cfg="standard", norm_cfg="layer_norm", functional_cfg="torch",
                 loss_functional_cfg="torch"):
        super().__init__()
        self.cfg = cfg
        linear_factory = factories.get_linear_factory(linear_cfg)
        norm_factory = factories.get_norm_factory(norm_cfg)
        norm_layer = lambda dim: norm_factory(dim, eps=cfg.eps)
        op_dict = factories.get_function_dict(functional_cfg)
        self.loss_ops = factories.get_function_dict(loss_functional_cfg)
        self.encoder = _Stack(cfg, cfg.encoder_layers, False, linear_factory, norm_layer, op_dict)
        self.decoder = _Stack(cfg, cfg.decoder_layers, True, linear_factory, norm_layer, op_dict)
        # the decoder's input and output embeddings are shared: the output projection is a layer of the
        # linear factory whose weight is the embedding table (transformer_decoder.py:455-463)
        self.decoder.output_projection = linear_factory(cfg.dim, cfg.vocab, bias=False)
        self.decoder.output_projection.weight = self.decoder.embed_tokens.weight

    def encode(self, src, src_lengths=None):
        """The encoder's output.  `src_lengths` (int64 [sentences]): the tokens behind a sentence's length are padding, which no other position
        attends to."""
        mask = None if src_lengths is None else _beyond(src_lengths, src.shape[1]).repeat_interleave(self.cfg.heads, 0)
        x = self.encoder.embed(src)
        for layer in self.encoder.layers:
            x = layer(x, self_mask=mask)
        return x

    def forward(self, src, prev_out):
        x = self.encode(src)
        future = self.decoder._future(prev_out.shape[1], src.device)
        y = self.decoder.embed(prev_out)
        for layer in self.decoder.layers:
            y = layer(y, x, future)
        return self.decoder.output_projection(y)

    @torch.no_grad()
    def generate(self, src, beam=5, max_len=200, *, src_lengths=None, min_len=1, length_penalty=1.0, eos=2):
        """Beam search (fairseq/sequence_generator.py:199-552, search.py:103-147): the `beam` best translations of each sentence.

        src [sentences, length], padded behind `src_lengths` where these are given.  At most `max_len` tokens come out, the end of
        sentence `eos` among them (forced at the last one, not before the `min_len`-th).  Returns (tokens [sentences, beam, n], scores
        [sentences, beam]), best first; a hypothesis' score is its log-probability over its length to the power of
        `length_penalty`, -inf (and padding alone) where there were fewer; tokens behind the end are padding.  A sentence that has its `beam`
        hypotheses keeps them while others of the batch go on: in a batch it gets what it gets alone, up to rounding.

        The source's keys and values are kept once for the beams of a sentence, which attend to them together; each beam's own go where
        the beam goes on."""
        cfg, ops, device = self.cfg, self.decoder.op_dict, src.device
        if not 1 <= min_len <= max_len or beam < 1 or 2 * beam > decoding.MAX_SELECTED:
            raise ValueError(f"generate needs 1 <= min_len <= max_len and up to {decoding.MAX_SELECTED // 2} beams")
        if eos == cfg.pad or not 0 <= eos < cfg.vocab or cfg.vocab < 3:
            raise ValueError(f"end of sentence {eos} with padding {cfg.pad} in a vocabulary of {cfg.vocab}")
        if src_lengths is not None and not bool(((src_lengths >= 1) & (src_lengths <= src.shape[1])).all()):
            raise ValueError(f"lengths must be from 1 to {src.shape[1]}")
        memory = self.encode(src, src_lengths)
        shared = [layer.encoder_attn.cache(memory) for layer in self.decoder.layers]
        G, H = src.shape[0], cfg.heads
        own = [tuple(torch.empty(G, beam, max_len, H, cfg.dim // H, dtype=memory.dtype, device=device) for _ in range(2)) for _ in self.decoder.layers]
        caches = [t for pair in own for t in pair]
        positions = self.decoder._positions(max_len, device)
        tokens = torch.full((G, beam, max_len), cfg.pad, device=device)
        last = torch.full((G, beam), eos, device=device)
        scores = torch.full((G, beam), float("-inf"), device=device)
        scores[:, 0] = 0.0
        best, best_tokens = torch.full((G, beam), float("-inf"), device=device), tokens.clone()
        # what may not be chosen: early, in between and at last
        banned = torch.zeros(3, cfg.vocab, dtype=torch.bool, device=device)
        banned[:, cfg.pad] = True
        banned[0, eos] = True
        banned[2] = True
        banned[2, eos] = False
        count = min(2 * beam, beam * cfg.vocab)
        rank = torch.arange(count, device=device)
        for t in range(max_len):
            x = ops["mul"](self.decoder.embed_scale, self.decoder.embed_tokens(last)) + positions[t]
            for layer, mine, ours in zip(self.decoder.layers, own, shared):
                x = layer.step(x, mine, t, ours, src_lengths)
            logits = self.decoder.output_projection(x)
            found, parents, chosen = _select(ops, logits, scores, count, banned[2 if t == max_len - 1 else 0 if t + 1 < min_len else 1])
            # the ends of sentences among the first `beam` are hypotheses; the best are kept
            ends = chosen == eos
            done = torch.where(ends & (rank < beam), found / (t + 1) ** length_penalty, float("-inf"))
            longer = tokens.gather(1, parents.unsqueeze(-1).expand(-1, -1, max_len))
            longer[:, :, t] = chosen
            best, at = (x[:, :beam] for x in torch.cat([best, done], 1).sort(dim=1, descending=True, stable=True))
            best_tokens = torch.cat([best_tokens, longer], 1).gather(1, at.unsqueeze(-1).expand(-1, -1, max_len))
            finished = (best > float("-inf")).all(1, keepdim=True)
            if t == max_len - 1 or bool(finished.all()):
                break
            # the first `beam` others go on; none of a finished sentence, which finds no more ends then
            go = (rank + count * ends).argsort(1)[:, :beam]
            scores, parents, last = (v.gather(1, go) for v in (found, parents, chosen))
            scores = scores.masked_fill(ends.gather(1, go) | finished, float("-inf"))
            _reorder(caches, parents, t + 1)
            _reorder([tokens], parents, t)
            tokens[:, :, t] = last
        best_tokens = best_tokens.masked_fill((best == float("-inf")).unsqueeze(-1), cfg.pad)
        return best_tokens[:, :, :t + 1], best

    def loss(self, src, prev_out, target, fused=False):
        """Label-smoothed negative log-likelihood summed over the target tokens.  `fused` takes the
        loss from the logits in one row kernel each way (pam_opt.label_smoothed_nll_loss): the same
        values up to the association of the row sums."""
        ops, cfg = self.loss_ops, self.cfg
        if fused:
            from . import pam_opt
            logits = self(src, prev_out).reshape(-1, cfg.vocab)
            return pam_opt.label_smoothed_nll_loss(logits, target.reshape(-1), cfg.label_smoothing, op_dict=ops)[0]
        lprobs = ops["log_softmax"](self(src, prev_out).reshape(-1, cfg.vocab), dim=-1)
        nll = -lprobs.gather(-1, target.reshape(-1, 1)).sum()
        smooth = -lprobs.sum()
        eps_i = ops["div"](cfg.label_smoothing, cfg.vocab - 1)
        return ops["mul"](nll, 1.0 - cfg.label_smoothing - eps_i) + ops["mul"](smooth, eps_i)

    def load_parameters(self, p):
        """Fills the model from the flat dictionary of `steps.transformer_params`."""
        attn = {"q": "q_proj", "k": "k_proj", "v": "v_proj", "out": "out_proj"}
        state = {"encoder.embed_tokens.weight": p["enc.embed"], "decoder.embed_tokens.weight": p["dec.embed"],
                 "decoder.output_projection.weight": p["dec.embed"]}
        for key, value in p.items():
            parts = key.split(".")
            if parts[1] == "embed":
                continue
            side = "encoder" if parts[0] == "enc" else "decoder"
            base = f"{side}.layers.{parts[1]}."
            kind = "weight" if parts[-1] == "w" else "bias"
            if parts[2] in ("self", "cross"):
                module = "self_attn" if parts[2] == "self" else "encoder_attn"
                state[f"{base}{module}.{attn[parts[3]]}.{kind}"] = value
            else:
                module = {"ln_self": "self_attn_layer_norm", "ln_cross": "encoder_attn_layer_norm",
                          "ln_ffn": "final_layer_norm", "fc1": "fc1", "fc2": "fc2"}[parts[2]]
                state[f"{base}{module}.{kind}"] = value
        self.load_state_dict({k: v.detach() for k, v in state.items()})
        return self


PAM_LINEAR_CFG = '{"subtype": "pam", "dkwargs": {"approx_bwd": true}}'
PAM_NORM_CFG = '{"subtype": "pam_ln", "dkwargs": {"approx_bwd": true}}'
PAM_FUNCTION_CFG = '{"type": "pam", "dkwargs": {"approx_bwd": true}}'


def pam_cfgs(approx_bwd=True):
    """The configuration strings of an all-PAM run (the forks' --linear-cfg / --norm-cfg /
    --functional-cfg / --loss-functional-cfg values), with the gradient mode filled in."""
    flag = "true" if approx_bwd else "false"
    return dict(linear=PAM_LINEAR_CFG.replace("true", flag), norm=PAM_NORM_CFG.replace("true", flag),
                function=PAM_FUNCTION_CFG.replace("true", flag))
