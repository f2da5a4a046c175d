"""A small spiking language model: how the operators of ``hip_linattn`` and ``hip_lm`` and the neurons of
``hip_lif`` run together, in training and one token at a time.

    x = norm(embed(tokens))                                  the residual stream, fp32
    each block:  o = lin_attn(q, k, v of z)                  mixes the tokens: a leaky matrix state a head
                 x, z = block_norm(x, Wo o, gate = Wg z)     norm, gate, residual scale, next norm
                 s = LIF(W1 z)                               hard-reset neurons: spikes over time
                 x, z = block_norm(x, W2 s)
    logits = z We^T                                          the embedding table again

Arrays are time-major, tokens [T, B].  Nothing looks ahead, so a sequence may be fed whole, in pieces or
token by token: ``forward(tokens, state)`` takes and returns the state (the matrix states and the neurons'
membranes), ``step`` is its form for one token.  ``loss`` is the distillation from a teacher's top
logits, the usual way to train spiking language models.

Training runs the exact scan layers with the surrogate gradient (``lif_auto``) from resting neurons and
returns no state.  Without gradients (``torch.no_grad``, or a call with a state, which has none) the serial
forward carries the membranes, and every call returns the state after it.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import hip_lif as L
from . import hip_linattn as LA
from . import hip_lm as LM

THETA, RESET, SURROGATE = 1.0, 0.0, 4.0


class Block(nn.Module):
    """One mixing layer and one layer of neurons.  dtype: of the mixing layer's operands (the neurons and
    the residual stream are fp32)."""

    def __init__(self, D, heads, dk, dv, neurons, beta=0.95, dtype=torch.float32):
        super().__init__()
        self.heads, self.dk, self.dv, self.beta, self.dtype = heads, dk, dv, beta, dtype
        self.qkv = nn.Linear(D, heads * (2 * dk + dv), bias=False)
        self.gate = nn.Linear(D, D, bias=False)
        self.out = nn.Linear(heads * dv, D, bias=False)
        self.up = nn.Linear(D, neurons, bias=False)
        self.down = nn.Linear(neurons, D, bias=False)
        for name in ("mix_post", "mix_pre", "spike_post", "spike_pre"):
            self.register_parameter(name, nn.Parameter(torch.ones(D)))
        self.mix_scale, self.spike_scale = (nn.Parameter(torch.full((D,), 0.5)) for _ in range(2))
        # half-lives from a few tokens to some hundred
        self.register_buffer("decay", 1 - torch.exp2(-torch.linspace(2, 9, heads)))

    def _split(self, z):
        h, dk, dv = self.heads, self.dk, self.dv
        q, k, v = F.linear(z, self.qkv.weight.to(self.dtype)).split([h * dk, h * dk, h * dv], -1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (h, dk)), v.unflatten(-1, (h, dv))

    def _mixed(self, x, z, o):
        y = F.linear(o.flatten(-2), self.out.weight.to(self.dtype))
        g = F.linear(z, self.gate.weight.to(self.dtype))
        return LM.block_norm(x, y, self.mix_post, self.mix_pre, gate=g, res_scale=self.mix_scale)

    def _spiked(self, x, s):
        y = F.linear(s.to(self.dtype), self.down.weight.to(self.dtype))
        return LM.block_norm(x, y, self.spike_post, self.spike_pre, res_scale=self.spike_scale)

    def forward(self, x, z, state=None):
        """x (fp32), z [T, B, D] -> x, z, the state after the last row (None with gradients).  state: (matrix
        states, membranes) or None for a start at rest."""
        T, B, _ = x.shape
        o, S = LA.lin_attn(*self._split(z), self.decay, s0=state and state[0], scale=self.dk ** -0.5)
        x, z = self._mixed(x, z, o)
        currents = self.up(z.float()).flatten(1)
        u = state[1] if state else currents.new_zeros(currents.shape[1])
        if T == 0:
            s = currents  # the neurons take one row at least
        elif torch.is_grad_enabled():
            s = L.lif_auto(currents, u, self.beta, THETA, RESET, SURROGATE)
        else:
            U, s = L.serial_forward(currents, self.beta, THETA, RESET, u)
            u = U[-1].clone()  # not a view that keeps all rows
        after = None if torch.is_grad_enabled() else (S, u)
        x, z = self._spiked(x, s.unflatten(1, (B, -1)))
        return x, z, after

    def step(self, x, z, state):
        """One token: x, z [B, D]; the matrix states are updated in place."""
        S, u = state
        o = LA.lin_attn_step(*self._split(z), self.decay, S, scale=self.dk ** -0.5)
        x, z = self._mixed(x, z, o)
        U, s = L.serial_forward(self.up(z.float()).view(1, -1), self.beta, THETA, RESET, u)
        x, z = self._spiked(x, s.view(x.shape[0], -1))
        return x, z, (S, U[0])


class SpikeLM(nn.Module):
    def __init__(self, vocab, D=256, layers=2, heads=4, dk=64, dv=64, neurons=512, beta=0.95,
                 dtype=torch.float32):
        super().__init__()
        self.D, self.dtype = D, dtype
        self.table = nn.Parameter(torch.randn(vocab, D) * D ** -0.5)
        self.start_post, self.start_pre = nn.Parameter(torch.ones(D)), nn.Parameter(torch.ones(D))
        self.blocks = nn.ModuleList(Block(D, heads, dk, dv, neurons, beta, dtype) for _ in range(layers))

    def state(self, B):
        """The state of B sequences before their first token."""
        like = self.table
        return [(like.new_zeros(B, b.heads, b.dk, b.dv), like.new_zeros(B * b.up.out_features)) for b in self.blocks]

    def _check_state(self, state, B, in_place=False):
        """Before anything is changed: a state of B sequences, whole."""
        def fits(t, shape):
            return torch.is_tensor(t) and tuple(t.shape) == shape and t.dtype == torch.float32 \
                and t.device == self.table.device

        if len(state) != len(self.blocks):
            raise ValueError(f"a state of {len(self.blocks)} blocks is needed, got {len(state)}")
        for i, (s, b) in enumerate(zip(state, self.blocks)):
            shapes = (B, b.heads, b.dk, b.dv), (B * b.up.out_features,)
            if s is None or len(s) != 2 or not all(fits(t, n) for t, n in zip(s, shapes)) \
                    or in_place and not s[0].is_contiguous():
                raise ValueError(f"block {i}: the state must be a matrix state {shapes[0]} and membranes {shapes[1]}, "
                                 f"as a call without gradients returns them")

    def _start(self, tokens):
        e = LM.embed(tokens, self.table, scale=self.D ** 0.5).to(self.dtype)
        return LM.block_norm(torch.zeros(e.shape, device=e.device), e, self.start_post, self.start_pre)

    def _logits(self, z):
        return F.linear(z, self.table.to(self.dtype))

    def forward(self, tokens, state=None):
        """tokens [T, B] -> logits [T, B, vocab], and the state after the last token (None with gradients).
        state: as returned (or ``state(B)``), to continue sequences, without gradients; None: from their
        start."""
        if state is not None:
            self._check_state(state, tokens.shape[1])
        with torch.set_grad_enabled(torch.is_grad_enabled() and state is None):
            x, z = self._start(tokens)
            after = []
            for i, block in enumerate(self.blocks):
                x, z, s = block(x, z, None if state is None else state[i])
                after.append(s)
            return self._logits(z), None if torch.is_grad_enabled() else after

    @torch.no_grad()
    def step(self, tokens, state):
        """One token of each sequence: tokens [B] -> logits [B, vocab]; `state` is updated in place."""
        self._check_state(state, tokens.shape[0], in_place=True)
        x, z = self._start(tokens)
        for i, block in enumerate(self.blocks):
            x, z, state[i] = block.step(x, z, state[i])
        return self._logits(z)

    def loss(self, tokens, top_values, top_index, temperature=1.0):
        """Mean distillation loss of tokens [T, B] against the teacher's top logits [T, B, K]."""
        logits, _ = self(tokens)
        return LM.distill_topk(logits, top_values, top_index, temperature).mean()
