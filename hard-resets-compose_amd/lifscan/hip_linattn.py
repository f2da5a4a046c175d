"""Linear attention with a decay for each head: a leaky integrator whose state is a matrix,

    S_t = beta*S_{t-1} + k_t v_t^T          o_t = scale * q_t^T S_t

the mixing layer of a spiking language model, next to the LIF membrane u = beta*u + x of
``hip_lif``.  Arrays are time-major as everywhere in this package: q [T, B, Hq, Dk], k [T, B, Hk, Dk],
v [T, B, Hv, Dv], o [T, B, H, Dv], states [B, H, Dk, Dv] in fp32.  Any strides are taken as they are
when the last axis is contiguous, so views of one projection, or ``x.transpose(0, 1)`` of a
batch-major array, are not copied.

  lin_attn        a prompt or a training step, with gradients for q, k, v and the first state
  lin_attn_step   one new token; the state is updated in place

No counterpart in the reference.  There is no fallback: every call runs the HIP kernels of
liblifscan_hip.so (linattn_kernels.hip) through the C++ operators of ``_ops_lm.cpp``, which check the
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
    (fp32, contiguous) is updated in place.  No gradients: train with lin_attn."""
    return _n.lm_ops().lin_attn_step(q, k, v, _decays(beta, q, k, v), state, scale)
