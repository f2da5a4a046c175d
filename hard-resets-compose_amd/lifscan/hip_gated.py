"""A gated linear recurrence: a leaky integrator u = beta*u + x, as the membranes of ``hip_lif`` without their
spikes, whose decay is another one for each channel and token,

    a_t = sigmoid(gate_t), or exp(min(gate_t, 0))
    h_t = a_t*h_{t-1} + (1 - a_t)*x_t, or + x_t

a mixing layer of a spiking language model next to the linear attention of ``hip_linattn``.  Arrays are
time-major as everywhere in this package: x, gate, h [T, B, D], states [B, D] in fp32.  Any strides are taken
as they are when the last axis is contiguous, so views of one projection are not copied.

  gated_scan       a prompt or a training step, with gradients for x, gate and the first state
  gated_scan_step  one new token; the state is updated in place

No counterpart in the reference.  There is no fallback: every call runs the HIP kernels of
liblifscan_hip.so (gated_kernels.hip) through the C++ operators of ``_ops_lm.cpp``, which check the
arguments and raise ValueError.
"""
from . import _native as _n

DECAYS = {"sigmoid": 0, "log": 1}  # LSH_DECAY_*


def _decay(name):
    if name not in DECAYS:
        raise ValueError(f"decay {name!r}: 'sigmoid' or 'log'")
    return DECAYS[name]


def gated_scan(x, gate, h0=None, starts=None, decay="sigmoid", mix=True):
    """The recurrence over a sequence -> (h [T, B, D], state after the last row [B, D] fp32).

    x, gate [T, B, D]: float32, bfloat16 or float16, one type.  decay: "sigmoid" (a = sigmoid(gate)) or "log"
    (a = exp(gate); a gate above 0 counts as 0 and gets no gradient).  mix: inputs weighed by 1 - a, or as
    they are.  h0: the fp32 state before the first row, or None (zeros).  starts: bool [T, B], where a sequence
    starts anew: the state before that row, h0 among them, is dropped, whatever it holds.  Sums are fp32
    throughout; h is rounded to the type of x once.  A decay below the smallest normal fp32 number is 0.

    A value that is not finite reaches its own row and, until a start, the later rows of its channel, and no
    others.  What it reaches is not finite, but may be NaN where the recurrence has an infinity."""
    return _n.lm_ops().gated_scan(x, gate, h0, starts, _decay(decay), bool(mix))


def gated_scan_step(x, gate, state, decay="sigmoid", mix=True):
    """One token: x, gate [B, D] -> h [B, D]; `state` [B, D] (fp32, contiguous) is updated in place.  x and gate
    that share memory with it are taken as they were before.  No gradients: train with gated_scan."""
    return _n.lm_ops().gated_scan_step(x, gate, state, _decay(decay), bool(mix))
