"""
Transformer decoder forward (aps/asr/transformer/decoder.py:16-186) on the HIP kernels: token
embedding + sinusoid in one launch, causal self attention and cross attention on the attention
kernels, every projection / feed-forward on the fp32 MFMA GEMM with bias / activation / residual
(and, for pre-norm layers, the LayerNorm) in its epilogue.

Parameter names and shapes are the reference's (`vocab_embed.weight`, `decoder.layers.N.self_attn.
in_proj_weight` ... `decoder.norm.*`, `output.weight`): nn.MultiheadAttention / nn.LayerNorm /
nn.Linear modules hold them, the forward path does not call them.  Teacher-forced forward and
`step` (with `pre_emb`).  Under autograd / in train() mode every link has a HIP backward
(aps_amd/grad_ops.py): the projections, LayerNorms, the causal self attention (the context-window form
of the general attention adjoint), the attention over the encoder output (aps_attention_cross_backward),
the token embedding, and every dropout of the reference's layer -- on the attention weights, behind
the two attentions and inside / behind the feed-forward -- as counter-based masks.
"""
from typing import Callable, Dict, Optional, Tuple

import torch as th
import torch.nn as nn
from torch.nn import MultiheadAttention

from aps_amd.asr.transformer.impl import _check_activation, get_activation_fn
from aps_amd.grad_ops import ScaleAddFn, dropout, dropout_active
from aps_amd.asr.transformer.pose import get_xfmr_pose
from aps_amd.nn_ops import (BEAM_MAX, PACKED_HEAD_DIMS, attention_core, attention_cross, attention_packed,
                            attention_paged, beam_reorder, beam_select, embedding_posenc, layernorm, linear,
                            paged_append, posenc_add)


class TransformerDncoderLayer(nn.Module):
    """decoder layer: causal self attention, attention over the encoder output, feed-forward;
    pre- or post-norm (decoder.py:16-99; the class name is the reference's spelling)"""

    def __init__(self, att_dim: int, nhead: int, feedforward_dim: int = 2048,
                 pre_norm: bool = False, att_dropout: float = 0.1, ffn_dropout: float = 0.1,
                 activation: str = "relu") -> None:
        super(TransformerDncoderLayer, self).__init__()
        self.pre_norm = pre_norm
        self.activation = _check_activation(activation)
        self.self_attn = MultiheadAttention(att_dim, nhead, dropout=att_dropout)
        self.multihead_attn = MultiheadAttention(att_dim, nhead, dropout=att_dropout)
        self.feedforward = nn.Sequential(nn.Linear(att_dim, feedforward_dim),
                                         get_activation_fn(activation), nn.Dropout(ffn_dropout),
                                         nn.Linear(feedforward_dim, att_dim),
                                         nn.Dropout(ffn_dropout))
        self.norm1 = nn.LayerNorm(att_dim)
        self.norm2 = nn.LayerNorm(att_dim)
        self.norm3 = nn.LayerNorm(att_dim)
        self.dropout1 = nn.Dropout(ffn_dropout)
        self.dropout2 = nn.Dropout(ffn_dropout)
        self.nhead = nhead
        # nn.MultiheadAttention's `dropout` (on the attention weights) as modules that follow train() /
        # eval() (no parameters: the state dict is the reference's)
        self.self_attn_drop = nn.Dropout(att_dropout)
        self.cross_attn_drop = nn.Dropout(att_dropout)

    def memory_kv(self, memory: th.Tensor) -> th.Tensor:
        """key | value projections of the encoder output, N x S x D -> N x S x 2D"""
        att = self.multihead_attn
        D = att.embed_dim
        return linear(memory, att.in_proj_weight[D:], att.in_proj_bias[D:])

    def run(self, tgt: th.Tensor, memory: th.Tensor, tgt_len: Optional[th.Tensor],
            mem_len: Optional[th.Tensor], memory_mask: Optional[th.Tensor] = None,
            self_attend: Optional[Callable[[th.Tensor], th.Tensor]] = None,
            memory_kv: Optional[th.Tensor] = None) -> th.Tensor:
        """batch-major: tgt N x T x D, memory N x S x D -> N x T x D; memory_mask T x S additive.
        self_attend: what takes the place of the causal self attention over tgt itself (N x T x 3D -> N x T x D,
        the attention over a cache); memory_kv: memory_kv(memory), formed once for many calls"""
        sa, ca = self.self_attn, self.multihead_attn
        D = sa.embed_dim
        n1, n2, n3 = self.norm1, self.norm2, self.norm3
        pre = self.pre_norm

        def post(x, norm):
            return x if pre else layernorm(x, norm.weight, norm.bias, norm.eps)

        def out_proj(ctx, proj, residual, drop):
            """residual + dropout(out_proj(ctx)): one GEMM with the residual in its epilogue unless
            the dropout is active (train() mode)"""
            if dropout_active(drop):
                return ScaleAddFn.apply(dropout(linear(ctx, proj.weight, proj.bias), drop), residual, 1.0)
            return linear(ctx, proj.weight, proj.bias, residual=residual)

        # self attention under the sub-sequence mask (prep_sub_mask): key j <= query i
        qkv = linear(tgt, sa.in_proj_weight, sa.in_proj_bias, ln=n1 if pre else None)
        if self_attend is not None:
            ctx = self_attend(qkv)
        else:
            ctx = attention_core(qkv, self.nhead, tgt_len, chunk_size=1, lctx=-1, rctx=0,
                                 dropout=self.self_attn_drop)
        tgt = post(out_proj(ctx, sa.out_proj, tgt, self.dropout1), n1)
        # attention over the encoder output
        q = linear(tgt, ca.in_proj_weight[:D], ca.in_proj_bias[:D], ln=n2 if pre else None)
        ctx = attention_cross(q, self.memory_kv(memory) if memory_kv is None else memory_kv, self.nhead, mem_len,
                              memory_mask, dropout=self.cross_attn_drop)
        tgt = post(out_proj(ctx, ca.out_proj, tgt, self.dropout2), n2)
        # feed-forward: Linear - activation - Dropout - Linear - Dropout
        up, down = self.feedforward[0], self.feedforward[3]
        h = linear(tgt, up.weight, up.bias, act=self.activation, ln=n3 if pre else None)
        if dropout_active(self.feedforward[2], self.feedforward[4]):
            h = dropout(linear(dropout(h, self.feedforward[2]), down.weight, down.bias),
                        self.feedforward[4])
            return post(ScaleAddFn.apply(h, tgt, 1.0), n3)
        return post(linear(h, down.weight, down.bias, residual=tgt), n3)

    def forward(self, tgt: th.Tensor, memory: th.Tensor, tgt_mask: Optional[th.Tensor] = None,
                memory_mask: Optional[th.Tensor] = None,
                tgt_key_padding_mask: Optional[th.Tensor] = None,
                memory_key_padding_mask: Optional[th.Tensor] = None) -> th.Tensor:
        """reference call convention: T x N x D, S x N x D -> T x N x D.  The kernels build the
        sub-sequence mask themselves; padding masks must be length masks (as the reference's are).
        `memory_mask` (boolean or additive, T x S) is taken in eval and under autograd / in train() with
        dropout alike (round 5: the attention adjoints carry additive mask tensors -- data, no gradient
        into them; the reference's own decoder never passes one, aps/asr/transformer/decoder.py:133-186)"""
        if memory_mask is not None and memory_mask.dtype == th.bool:
            # nn.MultiheadAttention's boolean attn_mask (True = not visible) as the additive form
            memory_mask = th.zeros(memory_mask.shape, device=memory_mask.device).masked_fill_(
                memory_mask, float("-inf"))
        tl = None if tgt_key_padding_mask is None else (~tgt_key_padding_mask).sum(-1)
        ml = None if memory_key_padding_mask is None else (~memory_key_padding_mask).sum(-1)
        out = self.run(tgt.transpose(0, 1).contiguous(), memory.transpose(0, 1).contiguous(), tl, ml,
                       memory_mask)
        return out.transpose(0, 1)


class _DecoderStack(nn.Module):
    """parameter layout of torch's nn.TransformerDecoder: `layers.N.*` and optional `norm.*`"""

    def __init__(self, layer_kwargs: Dict, num_layers: int, norm: Optional[nn.Module]) -> None:
        super(_DecoderStack, self).__init__()
        self.layers = nn.ModuleList(
            [TransformerDncoderLayer(**layer_kwargs) for _ in range(num_layers)])
        self.norm = norm


class TorchTransformerDecoder(nn.Module):
    """Transformer decoder with absolute position encodings (decoder.py:102-186)"""

    def __init__(self, vocab_size: int, pose_kwargs: Dict = {}, arch_kwargs: Dict = {},
                 num_layers: int = 6) -> None:
        super(TorchTransformerDecoder, self).__init__()
        att_dim = arch_kwargs["att_dim"]
        self.vocab_embed = nn.Embedding(vocab_size, att_dim)
        self.abs_pos_enc = get_xfmr_pose("abs", att_dim, **pose_kwargs)
        final_norm = nn.LayerNorm(att_dim) if arch_kwargs.get("pre_norm") else None
        self.decoder = _DecoderStack(arch_kwargs, num_layers, final_norm)
        self.output = nn.Linear(att_dim, vocab_size, bias=False)
        self.vocab_size = vocab_size

    def step(self, enc_out: th.Tensor, tgt_pad: th.Tensor, enc_len: Optional[th.Tensor] = None,
             tgt_len: Optional[th.Tensor] = None, pre_emb: Optional[th.Tensor] = None,
             out_idx: Optional[int] = None) -> Tuple[th.Tensor, th.Tensor]:
        """enc_out T x N x D, tgt_pad N x To (, pre_emb T' x N x D) -> (dec_out T'+To x N x V or
        N x V for `out_idx`, tgt_emb T'+To x N x D)  (decoder.py:128-166)"""
        pose = self.abs_pos_enc
        offset = 0 if pre_emb is None else pre_emb.shape[0]
        emb = embedding_posenc(self.vocab_embed.weight, tgt_pad, pose.div_term, float(pose.factor),
                               offset)  # N x To x D
        emb = dropout(emb, pose.dropout)  # (InputSinPosEncoding's dropout, pose.py:93-118)
        if pre_emb is not None:
            emb = th.cat([pre_emb.transpose(0, 1), emb], 1)
        memory = enc_out.transpose(0, 1).contiguous()
        x = emb
        for layer in self.decoder.layers:
            x = layer.run(x, memory, tgt_len, enc_len)
        norm = self.decoder.norm
        if out_idx is not None:
            x = x[:, out_idx]
        if norm is not None:  # the final LayerNorm rides inside the output projection
            out = linear(x, self.output.weight, None, ln=norm)
        else:
            out = linear(x, self.output.weight, None)
        return (out if out_idx is not None else out.transpose(0, 1)), emb.transpose(0, 1)

    def forward(self, enc_out: th.Tensor, enc_len: Optional[th.Tensor], tgt_pad: th.Tensor,
                tgt_len: Optional[th.Tensor]) -> th.Tensor:
        """enc_out N x T x D, tgt_pad N x To -> N x To x V (decoder.py:168-186)"""
        dec_out, _ = self.step(enc_out.transpose(0, 1), tgt_pad, enc_len=enc_len, tgt_len=tgt_len)
        return dec_out.transpose(0, 1)

    @th.no_grad()
    def beam_search(self, enc_out: th.Tensor, enc_len: Optional[th.Tensor], prompt: th.Tensor, eos: int,
                    beam: int = 8, max_len: int = 100) -> Tuple[th.Tensor, th.Tensor, th.Tensor]:
        """Search over a key / value cache: enc_out N x T x D, prompt N x P tokens every hypothesis begins with (sos,
        ...) -> (tokens N x beam x L, scores N x beam, lengths N x beam): the tokens behind the prompt, best
        hypothesis first, score = the sum of their log-probabilities, eos included in tokens and lengths
        (`max_len` tokens without one if none came); behind it eos.

        The prompt goes through `attention_packed` and into a paged cache; then a step is one token a
        hypothesis: `paged_append`, `attention_paged`, `beam_select`, `beam_reorder`.  A page holds one token,
        so a hypothesis' past is a row of slot numbers: taking over another's past copies that row, no
        keys or values.  The module must be in eval() mode (no dropout)."""
        if any(m.training for m in self.modules()):
            raise RuntimeError("beam_search: put the decoder into eval() mode, all of its modules")
        if prompt.dim() != 2 or enc_out.dim() != 3 or prompt.shape[0] != enc_out.shape[0] or \
                (enc_len is not None and enc_len.shape != enc_out.shape[:1]):
            raise RuntimeError(f"beam_search: enc_out {tuple(enc_out.shape)}, prompt {tuple(prompt.shape)}, enc_len "
                               f"{None if enc_len is None else tuple(enc_len.shape)}: one prompt and one length an utterance")
        N, P = prompt.shape
        dev, dim = enc_out.device, self.vocab_embed.embedding_dim
        layers = list(self.decoder.layers)
        heads = layers[0].nhead
        head_dim = dim // heads
        if head_dim not in PACKED_HEAD_DIMS:
            raise NotImplementedError(f"beam_search: heads of {head_dim}, the cache's attention takes {PACKED_HEAD_DIMS}")
        if N < 1 or P < 1 or max_len < 1 or not 1 <= beam <= min(self.vocab_size, BEAM_MAX) or \
                not 0 <= eos < self.vocab_size:
            raise RuntimeError(f"beam_search: {N} prompts of {P} tokens, {max_len} more, beam {beam} (1 .. {BEAM_MAX}), eos "
                               f"{eos}, {self.vocab_size} tokens")
        pose = self.abs_pos_enc
        memory = enc_out.contiguous()
        kvs = [layer.memory_kv(memory) for layer in layers]
        caches = [th.empty(2, N * P + N * beam * max_len, 1, heads, head_dim, device=dev, dtype=th.float32)
                  for _ in layers]

        def forward(tokens: th.Tensor, at: int, table: th.Tensor, cu: th.Tensor, lens: th.Tensor) -> th.Tensor:
            """tokens N x rows x new (their positions at, at + 1, ...) -> logits of the last, N rows x V"""
            _, rows, new = tokens.shape
            x = embedding_posenc(self.vocab_embed.weight, tokens.reshape(N * rows, new), pose.div_term,
                                 float(pose.factor), at).view(N, rows * new, dim)
            for layer, kv, cache in zip(layers, kvs, caches):
                def attend(qkv: th.Tensor) -> th.Tensor:
                    q, k, v = qkv.view(-1, 3, heads, head_dim).unbind(1)
                    paged_append(k, v, cache[0], cache[1], table, cu, lens)
                    ctx = attention_packed(q, k, v, cu) if at == 0 else \
                        attention_paged(q, cache[0], cache[1], table, cu, lens)
                    return ctx.view(N, rows * new, dim)

                x = layer.run(x, memory, None, enc_len, self_attend=attend, memory_kv=kv)
            x = x.view(N * rows, new, dim)[:, -1]
            return linear(x, self.output.weight, None, ln=self.decoder.norm)

        # the prompt: one row of slots an utterance
        table = th.zeros(N, P + max_len, dtype=th.int32, device=dev)
        table[:, :P] = th.arange(N * P, dtype=th.int32, device=dev).view(N, P)
        cu = th.arange(0, N * P + 1, P, dtype=th.int32, device=dev)
        logits = forward(prompt.view(N, 1, P), 0, table, cu, th.full((N,), P, dtype=th.int32, device=dev))
        scores, parent, token, done = beam_select(logits, th.zeros(N, 1, device=dev, dtype=th.float32), eos, beam=beam)
        (table,) = beam_reorder([table], parent)
        tokens = th.full((N * beam, max_len), eos, dtype=th.int64, device=dev)
        tokens[:, 0] = token.view(-1)
        lengths = th.ones(N * beam, dtype=th.int64, device=dev)
        cu = th.arange(N * beam + 1, dtype=th.int32, device=dev)
        lens = th.full((N * beam,), P, dtype=th.int32, device=dev)
        slots = N * P + th.arange(N * beam, dtype=th.int32, device=dev)
        for t in range(1, max_len):
            if t % 8 == 0 and bool(done.all()):  # (a look at the device every eighth step)
                break
            lens += 1
            table[:, P + t - 1] = slots + N * beam * (t - 1)
            logits = forward(token.view(N, beam, 1), P + t - 1, table, cu, lens)
            scores, parent, token, done_next = beam_select(logits, scores, eos, finished=done)
            table, tokens, lengths, done = beam_reorder([table, tokens, lengths, done.view(-1)], parent)
            tokens[:, t] = token.view(-1)
            lengths += ~done
            done = done_next
        tokens = tokens[:, :int(lengths.max())]
        return tokens.view(N, beam, -1), scores, lengths.view(N, beam)
