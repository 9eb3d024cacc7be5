"""Self-attention with a sliding window and a few first tokens that stay visible (sinks), for decoders of long sequences.

    window_attn_func(q [T, B, H, D], k, v [T, B, H_kv, D], window, sinks, softmax_scale, lengths) -> [T, B, H, D]
        position i sees j where j <= i and (j > i - window or j < sinks); differentiable in q, k and v
    WindowSelfMultiheadAttn(embed_dim, num_heads, window, sinks, num_kv_heads, cache_bits)
        projections around it; decodes step by step from a QuantizedKVCache

Work and memory grow with T * (window + sinks): there is no mask tensor and no [T, T] tensor. H is a multiple of H_kv (query
heads share key / value heads). lengths (integers [B] on the device): positions behind a sequence's length see nothing, are
seen by nobody, and have zero outputs and gradients. fp16 / bf16, head dimension 64 or 128, no dropout on the probabilities,
torch.jit.trace is refused.
"""
import math

import torch
from torch import nn
from torch.nn import Parameter

from .. import _lib as L
from ._autocast import cast_if_autocast_enabled, no_autocast
from .linear import linear_function
from .quantized_cache import QuantizedKVCache


def window_attn_func(q, k, v, window, sinks=0, softmax_scale=None, lengths=None):
    L.refuse_tracing("window attention")
    if not torch.is_autocast_enabled():             # (the context manager costs half of a short call)
        return L.host().window_attention(q, k, v, window, sinks, softmax_scale, lengths)
    q, k, v = cast_if_autocast_enabled(q, k, v)
    with no_autocast():
        return L.host().window_attention(q, k, v, window, sinks, softmax_scale, lengths)


class WindowSelfMultiheadAttn(nn.Module):
    """in_proj_weight [(H + 2 H_kv) D, E] (rows ordered queries, keys, values; then head, head_dim), out_proj_weight [E, H D]
    and their biases. Training and whole sequences: forward(inputs [T, B, E], lengths). Decoding: make_cache(), then
    forward(inputs, lengths, cache=cache) for the prompt (an empty cache; its attention sees the unquantised rows) and for every step
    of one or a few positions (attended to from the cache, these included)."""

    def __init__(self, embed_dim, num_heads, window, sinks=4, num_kv_heads=None, cache_bits=4):
        super().__init__()
        self.embed_dim, self.num_heads, self.num_kv_heads = embed_dim, num_heads, num_kv_heads or num_heads
        self.head_dim = embed_dim // num_heads
        assert self.head_dim * num_heads == embed_dim, "embed_dim must be divisible by num_heads"
        assert num_heads % self.num_kv_heads == 0, "num_heads must be divisible by num_kv_heads"
        self.window, self.sinks, self.cache_bits = window, sinks, cache_bits
        rows = (num_heads + 2 * self.num_kv_heads) * self.head_dim
        self.in_proj_weight = Parameter(torch.empty(rows, embed_dim))
        self.out_proj_weight = Parameter(torch.empty(embed_dim, embed_dim))
        self.in_proj_bias = Parameter(torch.empty(rows))
        self.out_proj_bias = Parameter(torch.empty(embed_dim))
        self.reset_parameters()

    def reset_parameters(self):
        std_ = math.sqrt(2.0 / (self.embed_dim + self.embed_dim))
        nn.init.normal_(self.in_proj_weight, 0.0, std_)
        nn.init.normal_(self.out_proj_weight, 0.0, std_)
        nn.init.constant_(self.in_proj_bias, 0.)
        nn.init.constant_(self.out_proj_bias, 0.)

    def make_cache(self, batch, capacity, dtype=None):
        """dtype: of the rows that will be appended and of what read() returns; by default the weights', and for weights in 32 bits
        autocast's (bf16 outside of it)."""
        w = self.in_proj_weight
        if dtype is None:
            dtype = w.dtype
            if dtype == torch.float32:
                dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled() else torch.bfloat16
        return QuantizedKVCache(batch, self.num_kv_heads, self.head_dim, capacity, self.cache_bits, dtype, w.device)

    def forward(self, inputs, lengths=None, cache=None):
        """inputs [T, B, E] -> [T, B, E]. lengths [B]: as in window_attn_func; with a cache, how many of the T positions are a
        sequence's own (prompts of several lengths)."""
        L.refuse_tracing("window attention")
        t, b, _ = inputs.shape
        lin = linear_function(inputs, self.in_proj_weight, self.in_proj_bias)
        if cache is None or cache.longest == 0:
            with no_autocast():
                context = L.host().window_attention_projection(lin, self.num_heads, self.num_kv_heads, self.window, self.sinks, None, lengths)
        if cache is not None:
            heads = lin.detach().view(t, b, -1, self.head_dim)
            q, k, v = heads.split((self.num_heads, self.num_kv_heads, self.num_kv_heads), dim=2)
            first = cache.longest == 0
            if not first and lengths is not None:
                raise RuntimeError("window attention: lengths go with the prompt, a decoding step has the same positions for every sequence")
            if torch.is_grad_enabled() and lin.requires_grad:
                raise RuntimeError("window attention: decoding from a quantised cache has no gradient, call it under torch.no_grad()")
            cache.append(k, v, lengths)
            if not first:
                context = cache.attend(q, self.window, self.sinks)
        return linear_function(context.view(t, b, self.embed_dim), self.out_proj_weight, self.out_proj_bias)
