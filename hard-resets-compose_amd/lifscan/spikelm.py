"""A small spiking language model: how the operators of ``hip_linattn``, ``hip_gated`` and ``hip_lm`` and the
neurons of ``hip_lif`` run together, in training and one token at a time.

    x = norm(embed(tokens))                                  the residual stream, fp32
    each block:  o = lin_attn(q, k, v of z)                  mixes the tokens: a leaky matrix state a head
                     (rotary: q, k = norm_rotate(q, k))          normed a head and turned by position before
                  or gated_scan(v, gate of z)                    or a leaky state a channel, its decay by token
                 x, z = block_norm(x, Wo o, gate = Wg z)     norm, gate, residual scale, next norm
                 s = LIF(W1 z)                               hard-reset neurons: spikes over time
                 x, z = block_norm(x, W2 s)
    logits = z We^T                                          the embedding table again

Arrays are time-major, tokens [T, B].  Nothing looks ahead, so a sequence may be fed whole, in pieces or
token by token: ``forward(tokens, state)`` takes and returns the state (the matrix states and the neurons'
membranes; with rotary also each sequence's next position), ``step`` is its form for one token.  ``loss`` is the
distillation from a teacher's top logits, the usual way to train spiking language models; ``likelihood_loss``
trains on the tokens themselves, and ``score`` tells the log probabilities of given tokens, how sure the model
was, and what else it would have said.

Training runs the exact scan layers with the surrogate gradient (``lif_auto``) from resting neurons and
returns no state.  Without gradients (``torch.no_grad``, or a call with a state, which has none) the serial
forward carries the membranes, and every call returns the state after it.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import hip_gated as G
from . import hip_lif as L
from . import hip_linattn as LA
from . import hip_lm as LM

THETA, RESET, SURROGATE = 1.0, 0.0, 4.0


class Block(nn.Module):
    """One mixing layer and one layer of neurons.  dtype: of the mixing layer's operands (the neurons and
    the residual stream are fp32).  mixer: "attention" or "gated" (heads*dv channels); rotary: queries and keys
    are normed and turned by their positions."""

    def __init__(self, D, heads, dk, dv, neurons, beta=0.95, dtype=torch.float32, mixer="attention", rotary=False):
        super().__init__()
        if mixer not in ("attention", "gated"):
            raise ValueError(f"mixer {mixer!r}: 'attention' or 'gated'")
        if rotary and mixer != "attention":
            raise ValueError("rotary is for mixer 'attention': a gated recurrence has no queries and keys")
        self.heads, self.dk, self.dv, self.beta, self.dtype = heads, dk, dv, beta, dtype
        self.mixer, self.rotary = mixer, rotary
        if mixer == "gated":
            self.vg = nn.Linear(D, heads * 2 * dv, bias=False)
            # decays of half-lives from a few tokens to some hundred
            self.gate_bias = nn.Parameter(torch.linspace(1.5, 6.0, heads * dv))
        else:
            self.qkv = nn.Linear(D, heads * (2 * dk + dv), bias=False)
        self.gate = nn.Linear(D, D, bias=False)
        self.out = nn.Linear(heads * dv, D, bias=False)
        self.up = nn.Linear(D, neurons, bias=False)
        self.down = nn.Linear(neurons, D, bias=False)
        for name in ("mix_post", "mix_pre", "spike_post", "spike_pre"):
            self.register_parameter(name, nn.Parameter(torch.ones(D)))
        self.mix_scale, self.spike_scale = (nn.Parameter(torch.full((D,), 0.5)) for _ in range(2))
        if mixer == "attention":
            # half-lives from a few tokens to some hundred
            self.register_buffer("decay", 1 - torch.exp2(-torch.linspace(2, 9, heads)))
        if rotary:
            self.q_norm, self.k_norm = nn.Parameter(torch.ones(dk)), nn.Parameter(torch.ones(dk))
            self.register_buffer("inv_freq", self._frequencies(), persistent=False)

    def _frequencies(self, device=None):
        return 10000.0 ** (torch.arange(self.dk // 2, dtype=torch.float64, device=device) * (-2.0 / self.dk))

    def _apply(self, fn, *args, **kw):
        super()._apply(fn, *args, **kw)
        if self.rotary:  # in 64 bits also where the module is cast to fewer
            self.inv_freq = self._frequencies(self.inv_freq.device)
        return self

    def state_form(self, B):
        """(shape, type) of each part of the state of B sequences: the mixing layer's state, the membranes, and
        with rotary the position of the next token."""
        mix = (B, self.heads * self.dv) if self.mixer == "gated" else (B, self.heads, self.dk, self.dv)
        form = [(mix, torch.float32), ((B * self.up.out_features,), torch.float32)]
        return form + [((B,), torch.int64)] if self.rotary else form

    def _split(self, z):
        h, dk, dv = self.heads, self.dk, self.dv
        q, k, v = F.linear(z, self.qkv.weight.to(self.dtype)).split([h * dk, h * dk, h * dv], -1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (h, dk)), v.unflatten(-1, (h, dv))

    def _heads(self, z, positions):
        q, k, v = self._split(z)
        if self.rotary:
            q, k = LA.norm_rotate(q, k, positions, self.inv_freq, self.q_norm, self.k_norm)
        return q, k, v

    def _gates(self, z):
        v, g = F.linear(z, self.vg.weight.to(self.dtype)).split(self.heads * self.dv, -1)
        return v, g + self.gate_bias.to(self.dtype)

    def _mixed(self, x, z, o):
        y = F.linear(o if self.mixer == "gated" else o.flatten(-2), self.out.weight.to(self.dtype))
        g = F.linear(z, self.gate.weight.to(self.dtype))
        return LM.block_norm(x, y, self.mix_post, self.mix_pre, gate=g, res_scale=self.mix_scale)

    def _spiked(self, x, s):
        y = F.linear(s.to(self.dtype), self.down.weight.to(self.dtype))
        return LM.block_norm(x, y, self.spike_post, self.spike_pre, res_scale=self.spike_scale)

    def forward(self, x, z, state=None):
        """x (fp32), z [T, B, D] -> x, z, the state after the last row (None with gradients).  state: as
        ``state_form`` tells, or None for a start at rest."""
        T, B, _ = x.shape
        if self.mixer == "gated":
            o, S = G.gated_scan(*self._gates(z), h0=state and state[0])
        else:
            at = torch.arange(T, device=x.device) if self.rotary else None
            if self.rotary and state:
                at = state[2] + at[:, None]
            o, S = LA.lin_attn(*self._heads(z, at), self.decay, s0=state and state[0], scale=self.dk ** -0.5)
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
        if after and self.rotary:
            after += (state[2] + T if state else torch.full((B,), T, device=x.device),)
        x, z = self._spiked(x, s.unflatten(1, (B, -1)))
        return x, z, after

    def step(self, x, z, state):
        """One token: x, z [B, D]; the mixing layer's state is updated in place."""
        S, u, *at = state
        if self.mixer == "gated":
            o = G.gated_scan_step(*self._gates(z), S)
        else:
            o = LA.lin_attn_step(*self._heads(z, *at or [None]), self.decay, S, scale=self.dk ** -0.5)
        x, z = self._mixed(x, z, o)
        U, s = L.serial_forward(self.up(z.float()).view(1, -1), self.beta, THETA, RESET, u)
        x, z = self._spiked(x, s.view(x.shape[0], -1))
        return x, z, (S, U[0], *(p + 1 for p in at))


class SpikeLM(nn.Module):
    def __init__(self, vocab, D=256, layers=2, heads=4, dk=64, dv=64, neurons=512, beta=0.95,
                 dtype=torch.float32, mixer="attention", rotary=False):
        super().__init__()
        self.D, self.dtype = D, dtype
        self.table = nn.Parameter(torch.randn(vocab, D) * D ** -0.5)
        self.start_post, self.start_pre = nn.Parameter(torch.ones(D)), nn.Parameter(torch.ones(D))
        self.blocks = nn.ModuleList(Block(D, heads, dk, dv, neurons, beta, dtype, mixer, rotary) for _ in range(layers))

    def state(self, B):
        """The state of B sequences before their first token."""
        dev = self.table.device
        return [tuple(torch.zeros(n, dtype=t, device=dev) for n, t in b.state_form(B)) for b in self.blocks]

    def _check_state(self, state, B, in_place=False):
        """Before anything is changed: a state of B sequences, whole."""
        def fits(t, form):
            return torch.is_tensor(t) and (tuple(t.shape), t.dtype) == form and t.device == self.table.device

        if len(state) != len(self.blocks):
            raise ValueError(f"a state of {len(self.blocks)} blocks is needed, got {len(state)}")
        for i, (s, b) in enumerate(zip(state, self.blocks)):
            form = b.state_form(B)
            if s is None or len(s) != len(form) or not all(fits(t, n) for t, n in zip(s, form)) \
                    or in_place and not s[0].is_contiguous():
                raise ValueError(f"block {i}: the state must be the mixing layer's {form[0][0]}, membranes {form[1][0]}"
                                 f"{' and positions ' + str(form[2][0]) if b.rotary else ''}, as a call without "
                                 f"gradients returns them")

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

    def score(self, tokens, targets, temperature=1.0, top=0):
        """What the model says about targets [T, B], the tokens that followed tokens [T, B] (-1: none) -> log
        probabilities and entropies [T, B], and with top > 0 the alternatives' log probabilities and ids
        [T, B, top].  With gradients where they are enabled."""
        logits, _ = self(tokens)
        return LM.token_logprobs(logits, targets, temperature, top)

    def likelihood_loss(self, tokens, targets):
        """Mean negative log probability of the targets [T, B] that are tokens of the vocabulary."""
        logp, _ = self.score(tokens, targets)
        there = (targets >= 0) & (targets < self.table.shape[0])
        return -logp.sum() / there.sum().clamp(min=1)
