"""Linear attention with a decay for each head: S_t = lambda S_(t-1) + k_t v_t^T, o_t = scale S_t^T q_t, lambda = exp(log_decay).

    linear_attn_func(q, k, v [T, B, H, D], log_decay [H], scale, lengths, state, return_state, state_out) -> [T, B, H, D] (and the last state)
        whole sequences, in chunks on the matrix cores; differentiable in q, k, v and state
    linear_attn_step(q, k, v, log_decay, state, state_out, scale, lengths) -> [T, B, H, D]
        the newest positions of a decoder: reads the state and writes it behind them
    LinearSelfMultiheadAttn(embed_dim, num_heads, qk_norm, log_decay)
        projections around them; decodes step by step from a LinearAttnState

A state is fp32 [B, H, D, D] (keys by values), all of a sequence that a decoder needs: work and memory of a step do not grow with its
length. log_decay: fp32 on the device, at most 0 (larger values count as 0), no gradient. scale: D^-0.5 by default. lengths
(integers [B] on the device, clamped to [0, T]): positions behind a sequence's length change nothing and have zero outputs and
gradients. fp16 / bf16, head dimension 64 or 128, as many heads of keys and values as of queries; torch.jit.trace is refused.
"""
import math

import torch
from torch import nn
from torch.nn import Parameter

from .. import _lib as L
from ._autocast import cast_if_autocast_enabled, no_autocast
from .linear import linear_function
from .qk_norm import qk_norm_rotary_func


def linear_attn_func(q, k, v, log_decay, scale=None, lengths=None, state=None, return_state=False, state_out=None):
    """-> out, or (out, state) with return_state. state: fp32 [B, H, D, D] in front of the first position (None: zeros). state_out: a
    contiguous tensor that the last state is written to, state itself if wanted (no gradient)."""
    L.refuse_tracing("linear attention")
    if torch.is_autocast_enabled():
        q, k, v = cast_if_autocast_enabled(q, k, v)
    out, last = L.host().linear_attention(q, k, v, log_decay, scale, lengths, state, return_state, state_out)
    return (out, last) if return_state else out


def linear_attn_step(q, k, v, log_decay, state, state_out=None, scale=None, lengths=None):
    """The recurrence itself, position by position, in fp32 (one position, or a few). state is written in place, or left alone with
    another tensor state_out to write; both contiguous. lengths: how many of the T positions are a sequence's own. Under autocast the
    rows take its type, the state stays in fp32."""
    L.refuse_tracing("linear attention")
    if torch.is_autocast_enabled():
        q, k, v = cast_if_autocast_enabled(q, k, v)
    return L.host().linear_attention_step(q, k, v, log_decay, state, state_out, scale, lengths)


class LinearAttnState:
    """What a decoder keeps of `batch` sequences: `state` (fp32 [batch, heads, head_dim, head_dim]) and how many positions went
    into it, `lengths` (int32 [batch] on the device). Prompts and steps write both in place, so a captured one goes on with them."""

    def __init__(self, batch, heads, head_dim, device="cuda"):
        self.state = torch.zeros(batch, heads, head_dim, head_dim, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)

    def reorder(self, index):
        """Sequence i becomes what sequence index[i] was (beam search); the number of sequences may change. The tensors are new ones."""
        self.state, self.lengths = self.state.index_select(0, index), self.lengths.index_select(0, index)


class LinearSelfMultiheadAttn(nn.Module):
    """in_proj_weight [3 H D, E] (rows ordered queries, keys, values; then head, head_dim), out_proj_weight [E, H D] and their biases;
    with qk_norm q_norm_weight and k_norm_weight [D] and positions from pos_emb. log_decay: H numbers; by default heads that remember
    from 2 to 2048 positions. Training and whole sequences: forward(inputs [T, B, E], lengths). Decoding: make_state(), then
    forward(inputs, lengths, state=state) for the prompt and for every step behind it."""

    # Positions up to which decoding runs the recurrence, which is in 32 bits throughout, where chunks round the state for their products. us on the
    # device, recurrence and chunk: 5 x 8 heads of 64 3.0 and 5.6 for one position, 4.3 and 5.6 for four, 6.2 and 5.6 for eight, 9.8 and 5.6
    # for 16; 128 x 32 heads of 128 86 and 92, 99 and 97, 121 and 99, 176 and 109.
    STEP = 8

    def __init__(self, embed_dim, num_heads, qk_norm=True, log_decay=None):
        super().__init__()
        self.embed_dim, self.num_heads, self.head_dim = embed_dim, num_heads, embed_dim // num_heads
        assert self.head_dim * num_heads == embed_dim, "embed_dim must be divisible by num_heads"
        self.in_proj_weight = Parameter(torch.empty(3 * embed_dim, embed_dim))
        self.out_proj_weight = Parameter(torch.empty(embed_dim, embed_dim))
        self.in_proj_bias = Parameter(torch.empty(3 * embed_dim))
        self.out_proj_bias = Parameter(torch.empty(embed_dim))
        self.qk_norm = qk_norm
        if qk_norm:
            self.q_norm_weight = Parameter(torch.empty(self.head_dim))
            self.k_norm_weight = Parameter(torch.empty(self.head_dim))
        if log_decay is None:
            log_decay = [-2.0 ** -(1.0 + 10.0 * h / max(1, num_heads - 1)) for h in range(num_heads)]
        assert len(log_decay) == num_heads, "one decay for each head"
        # as bits: in 32 bits whatever type the parameters are converted to
        bits = torch.tensor([float(d) for d in log_decay], dtype=torch.float32).view(torch.int32)
        self.register_buffer("log_decay_bits", bits, persistent=False)
        self.reset_parameters()

    def reset_parameters(self):
        std_ = math.sqrt(2.0 / (self.embed_dim + self.embed_dim))
        nn.init.normal_(self.in_proj_weight, 0.0, std_)
        nn.init.normal_(self.out_proj_weight, 0.0, std_)
        nn.init.constant_(self.in_proj_bias, 0.)
        nn.init.constant_(self.out_proj_bias, 0.)
        if self.qk_norm:
            nn.init.constant_(self.q_norm_weight, 1.)
            nn.init.constant_(self.k_norm_weight, 1.)

    def make_state(self, batch):
        return LinearAttnState(batch, self.num_heads, self.head_dim, self.in_proj_weight.device)

    @property
    def log_decay(self):
        return self.log_decay_bits.view(torch.float32)

    def forward(self, inputs, lengths=None, state=None, pos_emb=None):
        """inputs [T, B, E] -> [T, B, E]. lengths [B]: how many of the T positions are a sequence's own. pos_emb: (cos, sin) tables of
        positions (with qk_norm); with a state, positions go on from its lengths, and one behind the tables' last row takes that row
        (more positions in one call than the tables have are an error): the tables have to reach as far as decoding goes."""
        L.refuse_tracing("linear attention")
        t, b, _ = inputs.shape
        if self.qk_norm and pos_emb is None:
            raise RuntimeError("linear attention: qk_norm needs pos_emb, the tables (cos, sin) of positions")
        lin = linear_function(inputs, self.in_proj_weight, self.in_proj_bias)
        decay = self.log_decay
        if state is not None and torch.is_grad_enabled() and lin.requires_grad:
            raise RuntimeError("linear attention: decoding from a state has no gradient, call it under torch.no_grad()")
        q, k, v = lin.view(t, b, 3 * self.num_heads, self.head_dim).split(self.num_heads, dim=2)
        if self.qk_norm:
            if state is not None and lengths is None and t > pos_emb[0].shape[0]:
                raise RuntimeError(f"linear attention: positions 0 to {t - 1} of tables of {pos_emb[0].shape[0]} rows")
            positions = None if state is None else state.lengths
            q, k = qk_norm_rotary_func(q, k, self.q_norm_weight, self.k_norm_weight, *pos_emb, positions=positions)
        with no_autocast():
            if state is None:
                context = linear_attn_func(q, k, v, decay, lengths=lengths)
            else:
                if t <= self.STEP:
                    context = linear_attn_step(q, k, v, decay, state.state, lengths=lengths)
                else:
                    context = linear_attn_func(q, k, v, decay, lengths=lengths, state=state.state, state_out=state.state)
                state.lengths += t if lengths is None else lengths.clamp(0, t).to(state.lengths)
        return linear_function(context.view(t, b, self.embed_dim), self.out_proj_weight, self.out_proj_bias)
