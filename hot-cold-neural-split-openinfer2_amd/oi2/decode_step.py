"""The layer loop of DesdemonaEngine.forward (engine.py:406-442) over this
library's drop-in layers: per layer the attention with its residual
(engine.py:426-427), the next layer's cold fetch submitted from the
post-attention state (the lookahead, engine.py:431-436), then this layer's
FFN with the fetch it was given (engine.py:438).

Embedding, final norm and lm_head stay with the caller, as they are outside
the decode path this library replaces.  With the cold records resident in
HBM (or pinned memory) nothing in the loop waits on the host, so a caller may
capture a whole step in a CUDA/HIP graph.

The FFN side is either the drop-in layers (a list of SparseFFNLayer, any
batch) or a DecodeStack holding the same layers (one token): the stack runs
each layer as two kernels that also predict the next layer's cold set from
the layer's post-attention input, where the drop-in layers run a separate
predictor first.  Both give the same values.
"""
from __future__ import annotations

import torch

from .attention import GroupedQueryAttention
from .layer import SparseFFNLayer
from .paged import PagedKVCache, PagePlan
from .rotary import Rotary
from .stack import DecodeStack


class DecoderStep:
    def __init__(self, attention_layers: list[GroupedQueryAttention],
                 ffn_layers: "list[SparseFFNLayer] | DecodeStack"):
        n_ffn = ffn_layers.n_layers if isinstance(ffn_layers, DecodeStack) else len(ffn_layers)
        if len(attention_layers) != n_ffn:
            raise ValueError(f"{len(attention_layers)} attention layers but {n_ffn} FFN layers")
        self.attention_layers = attention_layers
        self.ffn_layers = ffn_layers

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, kv_caches=None):
        """x (B, T, H) fp16 (the embedded tokens); cos / sin the tables for
        the call's positions; kv_caches None or one (k, v) per layer.
        Returns (x after the last layer's FFN, the new caches), as the loop
        of engine.py:421-438 leaves them before the final norm."""
        if isinstance(self.ffn_layers, DecodeStack):
            return self._forward_stack(x, cos, sin, kv_caches)
        new_kv = []
        B, T, H = x.shape
        next_prefetch = self.ffn_layers[0].submit_cold_fetch(x)
        for li, (attn, ffn) in enumerate(zip(self.attention_layers, self.ffn_layers)):
            kv = kv_caches[li] if kv_caches else None
            resid = torch.empty_like(x)
            _, layer_kv = attn(x, cos, sin, kv, residual_out=resid)   # x + attention
            x = resid
            new_kv.append(layer_kv)
            this_prefetch = next_prefetch
            next_prefetch = (self.ffn_layers[li + 1].submit_cold_fetch(x)
                             if li + 1 < len(self.ffn_layers) else None)
            x = ffn(x, this_prefetch)
        return x, new_kv

    def _forward_stack(self, x, cos, sin, kv_caches):
        B, T, H = x.shape
        if B * T != 1:
            raise ValueError(f"a DecodeStack runs one token at a time, got batch {B} x {T}")
        stack = self.ffn_layers
        stack.predict(0, x.reshape(H))
        new_kv = []
        for li, attn in enumerate(self.attention_layers):
            kv = kv_caches[li] if kv_caches else None
            resid = torch.empty_like(x)
            _, layer_kv = attn(x, cos, sin, kv, residual_out=resid)   # x + attention
            new_kv.append(layer_kv)
            out = torch.empty_like(x)
            stack.layer(li, resid.reshape(H), out.reshape(H))         # FFN, and layer li + 1's set
            x = out
        return x, new_kv

    def forward_paged(self, x: torch.Tensor, cache: PagedKVCache, plan: PagePlan, rotary: Rotary) -> torch.Tensor:
        """The loop over a paged cache: x (tokens, H) fp16, the packed tokens of
        the step that ``cache.extend`` laid out in ``plan`` for requests of
        different lengths.  Layer li uses layer li of the cache.  The FFN takes
        the tokens as one batch, which shares a cold set: ``forward``'s, predicted
        from the mean over the rows' last tokens, of the rows that are taken
        and have tokens in the step (over a DecodeStack: one token).  Tokens
        without a position (of rejected rows, or past the step's last one) have
        no part in it, whatever they hold.  Returns x after the last layer's FFN."""
        if x.dim() != 2:
            raise ValueError(f"x must be (tokens, hidden), got {tuple(x.shape)}")
        N, H = x.shape
        if cache.n_layers < len(self.attention_layers):
            raise ValueError(f"a cache of {cache.n_layers} layers for {len(self.attention_layers)}")
        cache._tokens(x, cache._plan(plan))
        if N == 0:
            return x
        x = x.contiguous()
        stack = self.ffn_layers if isinstance(self.ffn_layers, DecodeStack) else None
        if stack is not None:
            if N != 1:
                raise ValueError(f"a DecodeStack runs one token at a time, got {N}")
            stack.predict(0, x.reshape(H))
        else:
            def fetch(ffn, x):      # one token: the query is that token's, whatever the plan says
                return ffn.submit_cold_fetch(x, plan) if N > 1 else ffn.submit_cold_fetch(x[None])
            prefetch = fetch(self.ffn_layers[0], x)
        for li, attn in enumerate(self.attention_layers):
            resid = torch.empty_like(x)
            attn.forward_paged(x, cache, plan, rotary, layer=li, residual_out=resid)
            if stack is not None:
                x = torch.empty_like(x)
                stack.layer(li, resid.reshape(H), x.reshape(H))
                continue
            this = prefetch
            if li + 1 < len(self.ffn_layers):
                prefetch = fetch(self.ffn_layers[li + 1], resid)
            x = self.ffn_layers[li](resid[None], this)[0]
        return x

    __call__ = forward
