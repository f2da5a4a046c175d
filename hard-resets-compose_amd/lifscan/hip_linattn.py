"""Linear attention with a decay for each head: a leaky integrator whose state is a matrix,

    S_t = beta*S_{t-1} + k_t v_t^T          o_t = scale * q_t^T S_t

the mixing layer of a spiking language model, next to the LIF membrane u = beta*u + x of
``hip_lif``.  Arrays are time-major as everywhere in this package: q [T, B, Hq, Dk], k [T, B, Hk, Dk],
v [T, B, Hv, Dv], o [T, B, H, Dv], states [B, H, Dk, Dv] in fp32.  Any strides are taken as they are
when the last axis is contiguous, so views of one projection, or ``x.transpose(0, 1)`` of a
batch-major array, are not copied.

  lin_attn        a prompt or a training step, with gradients for q, k, v and the first state
  lin_attn_step   one new token; the state is updated in place
  norm_rotate     before either: norms of queries and keys for each head and their rotation by position

No counterpart in the reference.  There is no fallback: every call runs the HIP kernels of
liblifscan_hip.so (linattn_kernels.hip, rotate_kernels.hip) through the C++ operators of ``_ops_lm.cpp``, which check the
arguments and raise ValueError.
"""
import torch

from . import _native as _n


def _decays(beta, *operands):
    """beta as a tensor: one value for each head of the state."""
    if torch.is_tensor(beta):
        return beta
    b = float(beta)
    if not 0.0 <= b < float("inf"):
        raise ValueError(f"beta={b}: a decay is finite and not negative")
    heads = max((x.shape[-2] for x in operands if x.dim() >= 2), default=1)
    return torch.full((heads,), b, dtype=torch.float32, device=operands[0].device)


def lin_attn(q, k, v, beta, s0=None, scale=1.0):
    """Linear attention over a sequence -> (o [T, B, H, Dv], state after the last row [B, H, Dk, Dv]).

    q [T, B, Hq, Dk], k [T, B, Hk, Dk], v [T, B, Hv, Dv]: float32, bfloat16 or float16, one type;
    widths 1 to 256.  beta: [H] decays on the device (finite, >= 0, of any float type), or one number for
    all heads; Hq, Hk and Hv divide H, and consecutive heads share one.  (A head that grows, beta > 1, is
    right as far as fp32 holds its state; above 4 it is walked row by row.)  s0: the fp32 state before the
    first row, or None (zeros).  A decay gets no gradient; a negative one on the device gives NaN.

    A value of v, or an element of s0, that is not finite reaches its own row and the later ones in its
    column, and no earlier row.  What it reaches is not finite, but which of NaN and infinity it is is
    not that of the recurrence: sums run in other orders, and 16-bit products take values in parts."""
    return _n.lm_ops().lin_attn(q, k, v, _decays(beta, q, k, v), s0, scale)


def lin_attn_step(q, k, v, beta, state, scale=1.0):
    """One token: q [B, Hq, Dk], k [B, Hk, Dk], v [B, Hv, Dv] -> o [B, H, Dv]; `state` [B, H, Dk, Dv]
    (fp32, contiguous) is updated in place.  Operands that share memory with it are taken as they were before.  No
    gradients: train with lin_attn."""
    return _n.lm_ops().lin_attn_step(q, k, v, _decays(beta, q, k, v), state, scale)


def norm_rotate(q, k, positions=None, inv_freq=None, q_weight=None, k_weight=None, eps=1e-6, pairs="halves"):
    """Queries and keys as they enter attention -> (q, k), contiguous, of the same shapes and type:

        y = x / sqrt(mean(x^2) + eps) * weight                           each head by itself
        (y_i, y_j) -> (y_i cos a - y_j sin a, y_i sin a + y_j cos a)     a = position * inv_freq[p] for pair p

    q [T, B, Hq, D], k [T, B, Hk, D], or [B, heads, D] for one token each: float32, bfloat16 or float16, one
    type; even D from 2 to 256.  positions: int64 or int32, [T], [T, B], or [B] for one token each; any size,
    also negative: angles are formed in 64 bits.  inv_freq: up to D/2 frequencies on the device (float64 keeps
    them as they are); the first 2*len columns rotate, the others pass, whatever they hold.  They come together;
    without them: no rotation.  pairs: "halves" (column p with p + len) or "neighbours" (2p with 2p + 1).
    q_weight, k_weight: [D] each; both None: no norm.
    Gradients for q, k and the weights."""
    if pairs not in ("halves", "neighbours"):
        raise ValueError(f"pairs {pairs!r}: 'halves' or 'neighbours'")
    return _n.lm_ops().norm_rotate(q, k, positions, inv_freq, q_weight, k_weight, eps, pairs == "neighbours")
