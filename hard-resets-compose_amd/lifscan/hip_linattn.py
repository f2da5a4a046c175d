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
liblifscan_hip.so (linattn_kernels.hip).
"""
import ctypes

import torch

from . import _native as _n

MAX_D = 256  # LSH_LINATTN_MAX_D


def _operand(x, name, dims, like=None):
    """x with its last axis contiguous, checked against the first operand."""
    if not torch.is_tensor(x) or x.dim() != dims:
        axes = "[T, B, heads, D]" if dims == 4 else "[B, heads, D]"
        raise ValueError(f"{name} must be a {dims}-D {axes} tensor")
    if like is None:
        if x.device.type != "cuda":
            raise ValueError(f"{name} must be a GPU (HIP) tensor")
        if x.dtype not in _n.DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16")
    elif x.device != like.device or x.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}")
    elif x.shape[:-2] != like.shape[:-2]:
        raise ValueError(f"{name} must have the leading axes {tuple(like.shape[:-2])}")
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _decays(beta, heads, device):
    """beta as [H] fp32 on the device: one value for each head of the state."""
    if not torch.is_tensor(beta):
        b = float(beta)
        if not 0.0 <= b < float("inf"):
            raise ValueError(f"beta={b}: a decay is finite and not negative")
        return torch.full((max(heads),), b, dtype=torch.float32, device=device)
    if beta.dim() != 1 or beta.device != device:
        raise ValueError(f"beta must be a number or a [heads] tensor on {device}")
    return beta.detach().to(torch.float32).contiguous()


def _state(s, shape, device, name):
    if not torch.is_tensor(s) or tuple(s.shape) != shape or s.dtype != torch.float32 or s.device != device:
        raise ValueError(f"{name} must be float32 {shape} on {device}")
    return s


def _args(q, k, v, beta, scale, dims):
    """The checked operands and the C argument block without its states and outputs."""
    q = _operand(q, "q", dims)
    k, v = _operand(k, "k", dims, q), _operand(v, "v", dims, q)
    Dk, Dv = q.shape[-1], v.shape[-1]
    if k.shape[-1] != Dk:
        raise ValueError(f"q and k must have the same width, got {Dk} and {k.shape[-1]}")
    if not (1 <= Dk <= MAX_D and 1 <= Dv <= MAX_D):
        raise ValueError(f"widths {Dk} and {Dv}: 1 to {MAX_D} are supported")
    heads = (q.shape[-2], k.shape[-2], v.shape[-2])
    beta = _decays(beta, heads, q.device)
    H = beta.numel()
    if H < 1 or any(h < 1 or H % h for h in heads):
        raise ValueError(f"{H} decays: the heads of q, k and v {heads} must divide them")
    a = _n.LinAttn()
    a.dtype, a.Dk, a.Dv = _n.DTYPES[q.dtype], Dk, Dv
    a.q_heads, a.k_heads, a.v_heads = heads
    a.T, a.B, a.H = q.shape[0] if dims == 4 else 1, q.shape[-3], H
    a.q, a.k, a.v, a.beta = q.data_ptr(), k.data_ptr(), v.data_ptr(), beta.data_ptr()
    a.q_sb, a.q_sh = q.stride(-3), q.stride(-2)
    a.k_sb, a.k_sh = k.stride(-3), k.stride(-2)
    a.v_sb, a.v_sh = v.stride(-3), v.stride(-2)
    if dims == 4:
        a.q_st, a.k_st, a.v_st = q.stride(0), k.stride(0), v.stride(0)
    a.scale = float(scale)
    return a, q, k, v, beta


def _forward(q, k, v, beta, s0, scale):
    a, q, k, v, beta = _args(q, k, v, beta, scale, 4)
    shape = (a.B, a.H, a.Dk, a.Dv)
    if s0 is not None:
        s0 = _state(s0, shape, q.device, "s0").contiguous()
        a.s0 = s0.data_ptr()
    o = torch.empty(a.T, a.B, a.H, a.Dv, dtype=q.dtype, device=q.device)
    s_end = torch.empty(shape, dtype=torch.float32, device=q.device)
    a.o, a.s_end = o.data_ptr(), s_end.data_ptr()
    lib = _n.lib()
    nbytes = lib.lsh_linattn_workspace(ctypes.byref(a))
    ws = _n.workspace(nbytes, q.device) if nbytes else None
    with _n.on_device(q):
        _n.check(lib.lsh_linattn_fwd(ctypes.byref(a), _n.ptr(ws), nbytes, _n.stream_of(q)), "lsh_linattn_fwd")
    return o, s_end, (q, k, v, beta, s0, ws)


def _backward(q, k, v, beta, s0, starts, scale, do, ds_end, want_ds0):
    a, q, k, v, beta = _args(q, k, v, beta, scale, 4)
    a.s0 = _n.ptr(s0)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    shape = (a.B, a.H, a.Dk, a.Dv)
    ds0 = torch.empty(shape, dtype=torch.float32, device=q.device) if want_ds0 else None
    if do is None:
        do = torch.zeros((), dtype=q.dtype, device=q.device).expand(a.T, a.B, a.H, a.Dv)
    do = _operand(do, "do", 4, q)
    if ds_end is not None:
        ds_end = _state(ds_end, shape, q.device, "ds_end").contiguous()
    lib = _n.lib()
    nbytes = lib.lsh_linattn_bwd_workspace(ctypes.byref(a))
    ws = _n.workspace(nbytes, q.device) if nbytes else None
    with _n.on_device(q):
        _n.check(lib.lsh_linattn_bwd(
            ctypes.byref(a), _n.ptr(starts), _n.ptr(do), do.stride(0), do.stride(1), do.stride(2), _n.ptr(ds_end),
            _n.ptr(dq), _n.ptr(dk), _n.ptr(dv), _n.ptr(ds0), _n.ptr(ws), nbytes, _n.stream_of(q)),
            "lsh_linattn_bwd")
    return dq, dk, dv, ds0


class LinAttnFn(torch.autograd.Function):
    """lin_attn with gradients for q, k, v and s0."""

    @staticmethod
    def forward(ctx, q, k, v, beta, s0, scale):
        o, s_end, kept = _forward(q, k, v, beta, s0, scale)
        ctx.save_for_backward(*kept)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, s_end

    @staticmethod
    def backward(ctx, do, ds_end):
        if do is None and ds_end is None:
            return None, None, None, None, None, None
        q, k, v, beta, s0, starts = ctx.saved_tensors  # starts: the states before the row segments
        dq, dk, dv, ds0 = _backward(q, k, v, beta, s0, starts, ctx.scale, do, ds_end, ctx.needs_input_grad[4])
        return dq, dk, dv, None, ds0, None


def lin_attn(q, k, v, beta, s0=None, scale=1.0):
    """Linear attention over a sequence -> (o [T, B, H, Dv], state after the last row [B, H, Dk, Dv]).

    q [T, B, Hq, Dk], k [T, B, Hk, Dk], v [T, B, Hv, Dv]: float32, bfloat16 or float16, one type;
    widths 1 to 256.  beta: [H] decays on the device (>= 0, of any float type), or one number for all
    heads; Hq, Hk and Hv divide H, and consecutive heads share one.  s0: the fp32 state before the
    first row, or None (zeros).  A decay gets no gradient."""
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in (q, k, v, s0, beta)):
        if torch.is_tensor(beta) and beta.requires_grad:
            raise ValueError("beta is a constant of lin_attn: it gets no gradient (pass beta.detach())")
        return LinAttnFn.apply(q, k, v, beta, s0, scale)
    return _forward(q, k, v, beta, s0, scale)[:2]


def lin_attn_step(q, k, v, beta, state, scale=1.0):
    """One token: q [B, Hq, Dk], k [B, Hk, Dk], v [B, Hv, Dv] -> o [B, H, Dv]; `state` [B, H, Dk, Dv]
    (fp32, contiguous) is updated in place.  No gradients: train with lin_attn."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        raise ValueError("lin_attn_step has no gradients: call it under torch.no_grad, or lin_attn")
    a, q, k, v, beta = _args(q, k, v, beta, scale, 3)
    _state(state, (a.B, a.H, a.Dk, a.Dv), q.device, "state")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    o = torch.empty(a.B, a.H, a.Dv, dtype=q.dtype, device=q.device)
    a.o = o.data_ptr()
    with _n.on_device(q):
        _n.check(_n.lib().lsh_linattn_step(ctypes.byref(a), _n.ptr(state), _n.stream_of(q)),
                 "lsh_linattn_step")
    return o
