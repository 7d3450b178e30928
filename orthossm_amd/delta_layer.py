"""A residual layer around the gated delta rule, for training and serving.

    h = layer_norm(x);  q, k, v, a, b = W_in h
    g = -e^{a_log} softplus(a + a_bias),  beta = sigmoid(b),  q, k of unit length
    y = x + W_out gated_delta(q, k, v, g, beta)

``forward`` takes sequences and carries the state from call to call; ``step``
takes one token a row and updates the states of a pool in place.  Both run the
gfx950 kernels (``layer_norm``, ``gated_delta``, ``gated_delta_step``); the
projections are torch's.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .delta import gated_delta, gated_delta_step
from .norm import layer_norm
from .synthetic import baseline_lambda


class GatedDeltaLayer(nn.Module):
    """``n_heads`` heads of ``value_dim`` values over states with ``head_dim``
    rows; queries and keys have ``n_qk_heads`` heads (n_heads by default)."""

    def __init__(self, d_model: int, n_heads: int = 8, head_dim: int | None = None, value_dim: int | None = None,
                 n_qk_heads: int | None = None, eps: float = 1e-5):
        super().__init__()
        n_qk_heads = n_heads if n_qk_heads is None else n_qk_heads
        if n_heads % n_qk_heads:
            raise ValueError(f"n_heads={n_heads} is not a multiple of n_qk_heads={n_qk_heads}")
        head_dim = d_model // n_heads if head_dim is None else head_dim
        value_dim = head_dim if value_dim is None else value_dim
        self.d_model, self.n_heads, self.n_qk_heads = d_model, n_heads, n_qk_heads
        self.head_dim, self.value_dim, self.eps = head_dim, value_dim, eps
        self.norm_weight = nn.Parameter(torch.ones(d_model))
        self.norm_bias = nn.Parameter(torch.zeros(d_model))
        self.splits = [n_qk_heads * head_dim, n_qk_heads * head_dim, n_heads * value_dim, n_heads, n_heads]
        self.in_proj = nn.Linear(d_model, sum(self.splits), bias=False)
        self.out_proj = nn.Linear(n_heads * value_dim, d_model, bias=False)
        # a = 0 gives the heads the decays of the framework's EMA, cycled
        lam = baseline_lambda(8)
        self.a_log = nn.Parameter(torch.log(-torch.log(lam)).repeat(-(-n_heads // 8))[:n_heads].clone())
        self.a_bias = nn.Parameter(torch.full((n_heads,), math.log(math.e - 1.0)))     # softplus(a_bias) = 1

    def new_state(self, slots: int, device=None) -> torch.Tensor:
        """Zero states [slots, heads, head_dim, value_dim], also a pool for ``step``."""
        return torch.zeros(slots, self.n_heads, self.head_dim, self.value_dim, dtype=torch.float32,
                           device=self.a_log.device if device is None else device)

    def _project(self, x: torch.Tensor):
        lead = x.shape[:-1]
        h = layer_norm(x, self.norm_weight, self.norm_bias, eps=self.eps)
        q, k, v, a, b = self.in_proj(h).split(self.splits, -1)
        q, k = (F.normalize(t.reshape(*lead, self.n_qk_heads, self.head_dim), dim=-1) for t in (q, k))
        g = -torch.exp(self.a_log) * F.softplus(a.float() + self.a_bias)
        return q, k, v.reshape(*lead, self.n_heads, self.value_dim), g, torch.sigmoid(b.float())

    def forward(self, x: torch.Tensor, state: torch.Tensor | None = None, lengths: torch.Tensor | None = None):
        """x [B,S,d_model]: (y [B,S,d_model], the state after it); ``lengths``
        [B] as in ``gated_delta`` (y is x past them)."""
        if x.dim() != 3 or x.shape[2] != self.d_model:
            raise ValueError(f"x must be [B,S,{self.d_model}], got {tuple(x.shape)}")
        out, state = gated_delta(*self._project(x), state_init=state, lengths=lengths, return_state=True)
        return x + self.out_proj(out.flatten(2)), state

    @torch.no_grad()
    def step(self, x: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor | None = None) -> torch.Tensor:
        """x [B,d_model], one token a row: y [B,d_model]; the states of
        ``pool`` are updated in place (``slots`` as in ``gated_delta_step``)."""
        if x.dim() != 2 or x.shape[1] != self.d_model:
            raise ValueError(f"x must be [B,{self.d_model}], got {tuple(x.shape)}")
        out = gated_delta_step(*self._project(x), pool, slots=slots)
        return x + self.out_proj(out.flatten(1))
