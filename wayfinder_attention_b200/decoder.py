"""Decoder-only LM harness around the Wayfinder attention op (prefill forward).

A compact restatement of the reference's ``TransformerLM`` for the one model
family on the hot path (``routing_attention/models/transformer.py:26-72``
block, ``:76-312`` model): token + learned position embeddings, pre-LN blocks
(``x + attn(ln1(x))``, ``x + ff(ln2(x))`` with a GELU FFN), final LayerNorm and
an LM head tied to the token embedding.  Parameter names match the reference
(``token_emb``, ``pos_emb``, ``blocks.N.attn.*``, ``blocks.N.ln1`` …), so its
``state_dict`` loads.  Only ``attention_type`` "learned_address" (this build's
kernels) and "dense_flash" (PyTorch SDPA, the dense baseline of
``models/attention.py:130-173``) are provided.

``fused_layers=True`` runs the rest of the blocks on this package's operators too
(``layer_norm``, and ``fused_linear`` with bias, GELU and residual in its epilogue),
forward and backward; ``score`` gives the log probability of each next token with
``token_logprobs``, which is what answers are scored and the model is trained by:

    lm = TransformerLM(vocab, fused_layers=True, dropout=0.0).to("cuda", torch.bfloat16)
    r = lm.score(input_ids, top_n=5)          # .logprob, .entropy, .top_logprobs, .top_tokens
    loss = -r.logprob.sum() / (input_ids[:, 1:] != lm.pad_token_id).sum()
    loss.backward()

``fused_ends=True`` runs the model's two ends, which share a weight, on ``token_embedding`` and
``linear_token_logprobs``: ``loss`` and ``score`` (without alternatives) then hold no logits,
whatever the vocabulary, and the tied weight's gradient is the sum of the two operators':

    lm = TransformerLM(vocab, fused_layers=True, fused_ends=True, dropout=0.0).to("cuda", torch.bfloat16)
    lm.loss(input_ids).backward()
"""

from __future__ import annotations

import functools
import inspect
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .attention import KeyVectorSparseAttention, LearnedAddressSparseAttention
from .embedding import token_embedding
from .layer_norm import layer_norm
from .linear import project, runs_as
from .linear_logprobs import linear_token_logprobs
from .token_logprobs import TokenLogprobs, token_logprobs


class DenseSDPAAttention(nn.Module):
    """Dense causal attention through ``F.scaled_dot_product_attention`` (``attention.py:130-173``)."""

    def __init__(self, d_model: int, n_heads: int, dropout: float = 0.1):
        super().__init__()
        self.n_heads = n_heads
        self.head_dim = d_model // n_heads
        self.scale = self.head_dim ** -0.5
        self.q_proj = nn.Linear(d_model, d_model)
        self.k_proj = nn.Linear(d_model, d_model)
        self.v_proj = nn.Linear(d_model, d_model)
        self.out_proj = nn.Linear(d_model, d_model)
        self.dropout_p = dropout
        self.fused_linear = False

    def forward(self, x: torch.Tensor, attn_mask: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None, **kwargs) -> torch.Tensor:
        B, T, D = x.shape
        q, k, v = (project(layer, x, self.fused_linear).view(B, T, self.n_heads, self.head_dim).transpose(1, 2)
                   for layer in (self.q_proj, self.k_proj, self.v_proj))
        out = F.scaled_dot_product_attention(
            q, k, v, is_causal=True, scale=self.scale, dropout_p=self.dropout_p if self.training else 0.0
        )
        return project(self.out_proj, out.transpose(1, 2).contiguous().view(B, T, D), self.fused_linear,
                       residual=residual)


def _norm(ln: nn.Module, x: torch.Tensor) -> torch.Tensor:
    if runs_as(ln, nn.LayerNorm) and len(ln.normalized_shape) == 1:
        if torch.is_autocast_enabled("cuda"):  # norms run in fp32 there
            weight, bias = (None if p is None else p.float() for p in (ln.weight, ln.bias))
            return layer_norm(x.float(), weight, bias, ln.eps)
        return layer_norm(x, ln.weight, ln.bias, ln.eps)
    return ln(x)


def _plain_embedding(emb: nn.Module) -> bool:
    """Whether a module is an ``nn.Embedding`` whose forward and gradient are ``token_embedding``'s."""
    return (runs_as(emb, nn.Embedding) and emb.padding_idx is None and emb.max_norm is None
            and not emb.scale_grad_by_freq and not emb.sparse)


@functools.lru_cache(maxsize=None)
def _names_residual(forward) -> bool:
    return "residual" in inspect.signature(forward).parameters


def _adds_residual(attn: nn.Module) -> bool:
    """Whether an attention module adds the block's residual itself.

    Its forward has to name it (**kwargs would drop it), and hooks have to see what they would see of it.
    """
    return _names_residual(type(attn).forward) and runs_as(attn, type(attn))


class TransformerBlock(nn.Module):
    def __init__(self, d_model: int, n_heads: int, d_ff: int, dropout: float, attention_module: nn.Module,
                 layer_idx: int = 0, fused_layers: bool = False):
        super().__init__()
        self.attn = attention_module
        self.fused_layers = fused_layers
        if fused_layers and hasattr(attention_module, "fused_linear"):
            attention_module.fused_linear = True
        self.layer_idx = layer_idx
        self.ln1 = nn.LayerNorm(d_model)
        self.ln2 = nn.LayerNorm(d_model)
        self.ff = nn.Sequential(
            nn.Linear(d_model, d_ff), nn.GELU(), nn.Dropout(dropout), nn.Linear(d_ff, d_model), nn.Dropout(dropout)
        )

    def forward(self, x: torch.Tensor, attn_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.fused_layers:
            return self._forward_fused(x, attn_mask)
        x = x + self.attn(self.ln1(x), attn_mask=attn_mask)
        return x + self.ff(self.ln2(x))

    def _forward_fused(self, x: torch.Tensor, attn_mask: Optional[torch.Tensor]) -> torch.Tensor:
        """The same block on ``layer_norm`` and ``fused_linear``, where its modules are what they stand for."""
        h = _norm(self.ln1, x)
        if _adds_residual(self.attn):
            x = self.attn(h, attn_mask=attn_mask, residual=x)
        else:
            x = x + self.attn(h, attn_mask=attn_mask)
        h = _norm(self.ln2, x)
        if not (runs_as(self.ff, nn.Sequential) and len(self.ff) == 5):
            return x + self.ff(h)
        up, act, drop_hidden, down, drop_out = self.ff
        if runs_as(act, nn.GELU) and act.approximate == "none":
            h = project(up, h, True, activation="gelu")
        else:
            h = act(project(up, h, True))
        h = drop_hidden(h)
        if runs_as(drop_out, nn.Dropout) and not (drop_out.training and drop_out.p > 0.0):
            return project(down, h, True, residual=x)
        return x + drop_out(project(down, h, True))


class TransformerLM(nn.Module):
    def __init__(
        self,
        vocab_size: int,
        d_model: int = 256,
        n_layers: int = 6,
        n_heads: int = 4,
        d_ff: int = 1024,
        max_seq_len: int = 512,
        dropout: float = 0.1,
        attention_type: str = "learned_address",
        routing_top_k: int = 32,
        address_dim: int = 32,
        retrieval_config: Optional[dict] = None,
        pad_token_id: int = 0,
        fused_layers: bool = False,
        fused_ends: bool = False,
    ):
        super().__init__()
        if attention_type not in ("learned_address", "key_vector", "dense_flash", "dense"):
            raise ValueError(f"attention_type {attention_type!r} is outside this build's scope")
        self.d_model = d_model
        self.max_seq_len = max_seq_len
        self.pad_token_id = pad_token_id
        self.fused_layers = fused_layers
        self.fused_ends = fused_ends
        self.token_emb = nn.Embedding(vocab_size, d_model)
        self.pos_emb = nn.Embedding(max_seq_len, d_model)
        self.dropout = nn.Dropout(dropout)
        self.blocks = nn.ModuleList()
        for i in range(n_layers):
            if attention_type == "learned_address":
                attn = LearnedAddressSparseAttention(
                    d_model, n_heads, routing_top_k, address_dim=address_dim, dropout=dropout,
                    retrieval_config=retrieval_config,
                )
            elif attention_type == "key_vector":
                attn = KeyVectorSparseAttention(d_model, n_heads, routing_top_k, dropout=dropout,
                                                retrieval_config=retrieval_config)
            else:
                attn = DenseSDPAAttention(d_model, n_heads, dropout)
            self.blocks.append(TransformerBlock(d_model, n_heads, d_ff, dropout, attn, layer_idx=i,
                                                fused_layers=fused_layers))
        self.ln_f = nn.LayerNorm(d_model)
        self.lm_head = nn.Linear(d_model, vocab_size, bias=False)
        self.lm_head.weight = self.token_emb.weight

    def _embed(self, input_ids: torch.Tensor) -> torch.Tensor:
        if (self.fused_ends and _plain_embedding(self.token_emb) and _plain_embedding(self.pos_emb)
                and self.token_emb.weight.dtype == self.pos_emb.weight.dtype):
            return token_embedding(input_ids, self.token_emb.weight, position_weight=self.pos_emb.weight)
        pos = torch.arange(input_ids.shape[1], device=input_ids.device).unsqueeze(0)
        return self.token_emb(input_ids) + self.pos_emb(pos)

    def _hidden(self, input_ids: torch.Tensor, attn_mask: Optional[torch.Tensor]) -> torch.Tensor:
        """What the head takes: the last norm's rows."""
        if attn_mask is None:
            attn_mask = input_ids != self.pad_token_id
        x = self.dropout(self._embed(input_ids))
        for block in self.blocks:
            x = block(x, attn_mask=attn_mask)
        return _norm(self.ln_f, x) if self.fused_layers else self.ln_f(x)

    def forward(self, input_ids: torch.Tensor, attn_mask: Optional[torch.Tensor] = None) -> dict:
        h = self._hidden(input_ids, attn_mask)
        return {"logits": project(self.lm_head, h, True) if self.fused_layers else self.lm_head(h)}

    def score(self, input_ids: torch.Tensor, attn_mask: Optional[torch.Tensor] = None, top_n: int = 0) -> TokenLogprobs:
        """How likely each next token is: ``TokenLogprobs`` of shape (B, T - 1) for ``input_ids`` (B, T).

        Entry t is about token t + 1 given the tokens up to t.  Padding (``pad_token_id``) gets
        log probability 0 and no gradient.  With ``fused_ends`` and no alternatives the logits are
        not rounded to the model's type, nor held.
        """
        # the last position has no next token; a whole row of logits a token keeps them uncopied
        following = torch.cat([input_ids[:, 1:], input_ids.new_full((input_ids.shape[0], 1), self.pad_token_id)], 1)
        # a hook on the model, or a subclass's forward, is about the logits
        plain = runs_as(self, type(self)) and type(self).forward is TransformerLM.forward
        if self.fused_ends and top_n == 0 and plain and runs_as(self.lm_head, nn.Linear):
            h, weight, bias = self._hidden(input_ids, attn_mask), self.lm_head.weight, self.lm_head.bias
            if torch.is_autocast_enabled("cuda"):  # the product in its type, as nn.Linear's is
                dtype = torch.get_autocast_dtype("cuda")
                h, weight, bias = (None if t is None else t.to(dtype) for t in (h, weight, bias))
            r = linear_token_logprobs(h, weight, following, bias=bias, ignore_index=self.pad_token_id)
            none = r.logprob.new_empty((*following.shape, 0))
            r = TokenLogprobs(r.logprob, r.entropy, none, none.long())
        else:
            logits = self(input_ids, attn_mask)["logits"]
            r = token_logprobs(logits, following, top_n=top_n, ignore_index=self.pad_token_id)
        return TokenLogprobs(*(t[:, :-1] for t in r))

    def loss(self, input_ids: torch.Tensor, attn_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Mean cross entropy of the next tokens, padding left out (0 where there is nothing else), in float32."""
        count = (input_ids[:, 1:] != self.pad_token_id).sum()
        return -self.score(input_ids, attn_mask).logprob.sum() / count.clamp_min(1)
