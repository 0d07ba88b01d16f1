# -*- coding: utf-8 -*-
"""Linear attention as a sequence layer beside ``SRU``.

``SRU`` keeps one number of state for each hidden unit; this layer keeps a width x width matrix for each head, decayed by
a gate of the token: S_t = exp(g_t) S_{t-1} + k_t^T v_t, o_t = q_t S_t / sqrt(width).  It is called like an ``SRU`` layer,
``h, state = layer(x)`` with ``x (len, batch, n_in)``, goes on from a state, and takes single tokens with ``step``.  Queries
and keys of every head are RMS-normalised and turned by the token's positions on several axes (for the (pixel, word)
sequence n = s*L + t of the multimodal SRU: ``ops.map_positions``), so that the layer sees where in the map a token is.

The projections are library GEMMs; everything between them runs in libdmn_hip.so (ops.head_norm_rotary,
ops.linear_attention, ops.linear_attention_step).  No counterpart in the reference.
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops


class LinearAttention(nn.Module):
    """``layer = LinearAttention(n_in, hidden, num_heads); h, state = layer(x, state, positions, lengths)``.

    * ``num_heads``: heads of the state; ``num_qk_heads`` (a divisor, default all): query and key heads, each shared by
      ``num_heads // num_qk_heads`` value heads.  hidden is num_heads heads of at most 128 columns.
    * ``sections``: pairs of every head that each position axis turns, () for a layer without positions.
    * float32, bfloat16 or float16 parameters and inputs; the gate's bias (``layer.bfloat16()`` and the like leave it alone), the
      decays and the state are float32.  The gate's product is rounded to the layer's type like every projection, then joined
      with its bias in float32.
    * parameters: ``weight (n_in, (2*num_qk_heads + num_heads) * width)`` = [q | k | v], ``gate (n_in, num_heads)``,
      ``gate_bias (num_heads)``, ``q_norm``, ``k_norm (width)``, ``out (hidden, hidden)``.
    """

    DECAY_SCALE = 1.0 / 16           # of the gate's log sigmoid: a decay of about 0.96 a token where the gate is at 0

    def __init__(self, input_size, hidden_size, num_heads, num_qk_heads=None, sections=(), base=10000.0, eps=1e-6):
        super().__init__()
        num_qk_heads = num_heads if num_qk_heads is None else num_qk_heads
        if hidden_size % num_heads or num_heads % num_qk_heads:
            raise ValueError("LinearAttention: hidden_size %d must be a multiple of num_heads %d, and that of num_qk_heads %d"
                             % (hidden_size, num_heads, num_qk_heads))
        self.n_in, self.n_out, self.heads, self.qk_heads = input_size, hidden_size, num_heads, num_qk_heads
        self.width = hidden_size // num_heads
        if self.width > ops.LINEAR_ATTENTION_MAX_WIDTH:
            raise ValueError("LinearAttention: heads of at most %d columns, got %d" % (ops.LINEAR_ATTENTION_MAX_WIDTH, self.width))
        self.sections, self.base, self.eps = tuple(sections), float(base), float(eps)
        self.weight = nn.Parameter(torch.empty(input_size, (2 * num_qk_heads + num_heads) * self.width))
        self.gate = nn.Parameter(torch.empty(input_size, num_heads))
        self.gate_bias = nn.Parameter(torch.empty(num_heads, dtype=torch.float32))
        self.q_norm = nn.Parameter(torch.empty(self.width))
        self.k_norm = nn.Parameter(torch.empty(self.width))
        self.out = nn.Parameter(torch.empty(hidden_size, hidden_size))
        self.init_weight()

    def init_weight(self):
        with torch.no_grad():
            for w in (self.weight, self.gate, self.out):
                val = math.sqrt(3.0 / w.shape[0])
                w.uniform_(-val, val)
            self.gate_bias.zero_()
            self.q_norm.fill_(1.0)
            self.k_norm.fill_(1.0)

    def _apply(self, fn, recurse=True):
        """Device moves and conversions; a conversion to 16 bits leaves the gate's bias in float32, where small updates of a
        decay that is close to 1 are not lost."""
        bias, grad = self.gate_bias.data, self.gate_bias.grad
        grad = None if grad is None else grad.data         # what a conversion in place does not reach
        super()._apply(fn, recurse)
        if self.gate_bias.dtype in (torch.bfloat16, torch.float16) and bias.dtype == torch.float32:
            self.gate_bias.grad = None
            self.gate_bias.data = bias.to(self.gate_bias.device)
            if grad is not None:
                self.gate_bias.grad = grad.to(self.gate_bias.device)
        return self

    def _product(self, x, w):
        if torch.is_grad_enabled() or not x.shape[0]:
            return x.mm(w)
        return ops.tuned_matmul(x, w, any_rows=True)     # inference: BLAS library chosen per shape, prompts' lengths in powers of two

    def _heads(self, x, positions):
        """q, k, v (T, B, heads, width) and the log decays (T, B, heads) of x (T, B, n_in)."""
        T, B = x.shape[:2]
        rows = x.reshape(T * B, self.n_in)
        n = self.qk_heads * self.width
        qkv = self._product(rows, self.weight).view(T, B, self.weight.shape[1])
        q, k, v = qkv.split([n, n, self.n_out], -1)
        g = F.logsigmoid(self._product(rows, self.gate).view(T, B, self.heads).float() + self.gate_bias.float()) * self.DECAY_SCALE
        q, k = ops.head_norm_rotary(q.view(T, B, self.qk_heads, self.width), k.view(T, B, self.qk_heads, self.width), self.q_norm,
                                    self.k_norm, positions, self.sections, self.base, self.eps)
        return q, k, v.view(T, B, self.heads, self.width), g

    def forward(self, input, state=None, positions=None, lengths=None):
        """input (T, B, n_in) -> h (T, B, hidden) and the state (B, heads, width, width) after the last token.
        positions (T, B, axes) or (T, axes); lengths (B,): tokens of each sample, rows of h behind them are zero."""
        if input.dim() != 3 or input.shape[2] != self.n_in:
            raise ValueError("LinearAttention expects (len, batch, %d), got %s" % (self.n_in, tuple(input.shape)))
        T, B = input.shape[:2]
        q, k, v, g = self._heads(input, positions)
        o, state = ops.linear_attention(q, k, v, g, state, lengths)
        return self._product(o.view(T * B, self.n_out), self.out).view(T, B, self.n_out), state

    @torch.no_grad()
    def step(self, input, state, positions=None):
        """One token (inference): input (B, n_in), state (B, heads, width, width) float32, updated in place; positions
        (B, axes).  Returns h (B, hidden)."""
        if input.dim() != 2 or input.shape[1] != self.n_in:
            raise ValueError("LinearAttention.step expects (batch, %d), got %s" % (self.n_in, tuple(input.shape)))
        q, k, v, g = self._heads(input.unsqueeze(0), None if positions is None else positions.unsqueeze(0))
        o = ops.linear_attention_step(q[0], k[0], v[0], g[0], state)
        return self._product(o.view(-1, self.n_out), self.out)
