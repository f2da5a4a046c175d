"""The row operators of a spiking language model on MI355X: what stands between its neurons
(``hip_lif``), its mixing layers (``hip_linattn``) and its matrix products.

  block_norm    the norm after a block, its gate and residual scale, and the norm before the next block
  embed         embedding lookup with scaling; the table's gradient sums by token, in position order
  distill_topk  the loss against a teacher's top logits

Tensors are float32, bfloat16 or float16; sums and statistics are fp32 and every result is rounded to
its tensor's type once.  Every operator is deterministic (no floating-point atomics).  No counterpart
in the reference.  There is no fallback: every call runs the HIP kernels of liblifscan_hip.so.
"""
import ctypes

import torch

from . import _native as _n

GATES = {None: 0, "silu": 1, "sigmoid": 2}  # LSH_GATE_*
MAX_D = 16384   # LSH_BLOCK_NORM_MAX_D
MAX_K = 4096    # LSH_DISTILL_MAX_K


def _tensor(x, name, like=None):
    if not torch.is_tensor(x):
        raise ValueError(f"{name} must be a tensor")
    if like is None:
        if x.device.type != "cuda":
            raise ValueError(f"{name} must be a GPU (HIP) tensor")
        if x.dtype not in _n.DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16")
    elif x.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")
    return x


def _wants_grad(*xs):
    return torch.is_grad_enabled() and any(torch.is_tensor(x) and x.requires_grad for x in xs)


# ------------------------------------------------------------------------- norms of a block
def _channel(w, D, like, name):
    """A per-channel parameter as [D] fp32 on the device (the cast is differentiable)."""
    if not torch.is_tensor(w) or w.device != like.device or tuple(w.shape) != (D,) or w.dtype not in _n.DTYPES:
        raise ValueError(f"{name} must be a float [{D}] tensor on {like.device}")
    return w.to(torch.float32).contiguous()


def _bn_args(x, y, gate, w_post, w_pre, scale, scale1, eps, act):
    a = _n.BlockNorm()
    a.x_dtype, a.dtype, a.act, a.D = _n.DTYPES[x.dtype], _n.DTYPES[y.dtype], act, x.shape[-1]
    a.rows = x.numel() // a.D
    a.x, a.y, a.gate = x.data_ptr(), y.data_ptr(), _n.ptr(gate)
    a.w_post, a.w_pre, a.scale = w_post.data_ptr(), w_pre.data_ptr(), _n.ptr(scale)
    a.scale1, a.eps = scale1, eps
    return a


def _bn_forward(x, y, gate, w_post, w_pre, scale, scale1, eps, act):
    a = _bn_args(x, y, gate, w_post, w_pre, scale, scale1, eps, act)
    x_new, z = torch.empty_like(x), torch.empty_like(y)
    with _n.on_device(x):
        _n.check(_n.lib().lsh_block_norm_fwd(ctypes.byref(a), _n.ptr(x_new), _n.ptr(z), _n.stream_of(x)),
                 "lsh_block_norm_fwd")
    return x_new, z


class BlockNormFn(torch.autograd.Function):
    """block_norm with gradients; x_new is computed again in the backward, so nothing is kept but the
    operands."""

    @staticmethod
    def forward(ctx, x, y, gate, w_post, w_pre, scale, scale1, eps, act):
        ctx.save_for_backward(x, y, gate, w_post, w_pre, scale)
        ctx.cfg = (scale1, eps, act)
        ctx.set_materialize_grads(False)
        return _bn_forward(x, y, gate, w_post, w_pre, scale, scale1, eps, act)

    @staticmethod
    def backward(ctx, gx, gz):
        if gx is None and gz is None:
            return (None,) * 9
        x, y, gate, w_post, w_pre, scale = ctx.saved_tensors
        need = ctx.needs_input_grad
        a = _bn_args(x, y, gate, w_post, w_pre, scale, *ctx.cfg)
        gx = gx.contiguous() if gx is not None else None
        gz = gz.contiguous() if gz is not None else None
        dx, dy = torch.empty_like(x), torch.empty_like(y)
        dgate = torch.empty_like(gate) if need[2] else None
        dw_post, dw_pre, dscale = (torch.empty_like(w) if n else None
                                   for w, n in ((w_post, need[3]), (w_pre, need[4]), (scale, need[5])))
        lib = _n.lib()
        nbytes = lib.lsh_block_norm_bwd_workspace(ctypes.byref(a))
        ws = _n.workspace(nbytes, x.device)
        with _n.on_device(x):
            _n.check(lib.lsh_block_norm_bwd(
                ctypes.byref(a), _n.ptr(gx), _n.ptr(gz), _n.ptr(dx), _n.ptr(dy), _n.ptr(dgate),
                _n.ptr(dw_post), _n.ptr(dw_pre), _n.ptr(dscale), _n.ptr(ws), nbytes, _n.stream_of(x)),
                "lsh_block_norm_bwd")
        return (dx if need[0] else None, dy if need[1] else None, dgate, dw_post, dw_pre, dscale, None,
                None, None)


def block_norm(x, y, w_post, w_pre, gate=None, res_scale=1.0, eps=1e-6, act="silu"):
    """The end of one block and the start of the next, rows along the last axis -> (x_new, z):

        n = y / sqrt(mean(y^2) + eps) * w_post          the block's output y, normalised
        x_new = x + res_scale * act(gate) * n           the residual stream
        z = x_new / sqrt(mean(x_new^2) + eps) * w_pre   the next block's input

    x (the residual stream) is float32 or has y's type; y and gate have one type.  w_post, w_pre: [D].
    gate: like y, or None (no gate); act: "silu" or "sigmoid".  res_scale: a number, or a [D] tensor
    with its own gradient."""
    x, y = _tensor(x, "x"), _tensor(y, "y")
    if x.dim() < 1 or x.shape != y.shape or x.device != y.device:
        raise ValueError(f"x and y must have one shape and device, got {tuple(x.shape)} and {tuple(y.shape)}")
    if x.dtype not in (torch.float32, y.dtype):
        raise ValueError(f"x must be float32 or {y.dtype}")
    D = x.shape[-1]
    if not 1 <= D <= MAX_D:
        raise ValueError(f"{D} channels: 1 to {MAX_D} are supported")
    if gate is not None and (_tensor(gate, "gate", x).shape != y.shape or gate.dtype != y.dtype):
        raise ValueError(f"gate must be {y.dtype} {tuple(y.shape)}")
    if act not in GATES or act is None:
        raise ValueError(f"act {act!r}: 'silu' or 'sigmoid'")
    if not eps >= 0:
        raise ValueError(f"eps={eps} must not be negative")
    w_post, w_pre = _channel(w_post, D, x, "w_post"), _channel(w_pre, D, x, "w_pre")
    scale, scale1 = (_channel(res_scale, D, x, "res_scale"), 0.0) if torch.is_tensor(res_scale) else \
        (None, float(res_scale))
    x, y, gate = x.contiguous(), y.contiguous(), gate.contiguous() if gate is not None else None
    args = (x, y, gate, w_post, w_pre, scale, scale1, float(eps), GATES[act] if gate is not None else 0)
    return BlockNormFn.apply(*args) if _wants_grad(x, y, gate, w_post, w_pre, scale) else _bn_forward(*args)


# ------------------------------------------------------------------------- embedding
def _embed_forward(tokens, weight, scale, pad):
    out = torch.empty(*tokens.shape, weight.shape[1], dtype=weight.dtype, device=weight.device)
    with _n.on_device(weight):
        _n.check(_n.lib().lsh_embed_fwd(
            _n.DTYPES[weight.dtype], _n.ptr(tokens), _n.ptr(weight), _n.ptr(out), tokens.numel(),
            weight.shape[0], weight.shape[1], pad, scale, _n.stream_of(weight)), "lsh_embed_fwd")
    return out


class EmbedFn(torch.autograd.Function):
    """embed with the table's gradient."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, pad):
        ctx.save_for_backward(tokens)
        ctx.cfg = (weight.shape, weight.dtype, scale, pad)
        return _embed_forward(tokens, weight, scale, pad)

    @staticmethod
    def backward(ctx, dout):
        (tokens,) = ctx.saved_tensors
        (V, D), dtype, scale, pad = ctx.cfg
        dout = dout.contiguous()
        dw = torch.empty(V, D, dtype=dtype, device=dout.device)
        lib = _n.lib()
        nbytes = lib.lsh_embed_bwd_workspace(tokens.numel(), V)
        ws = _n.workspace(nbytes, dout.device)
        with _n.on_device(dout):
            _n.check(lib.lsh_embed_bwd(
                _n.DTYPES[dtype], _n.ptr(tokens), _n.ptr(dout), _n.ptr(dw), tokens.numel(), V, D, pad, scale,
                _n.ptr(ws), nbytes, _n.stream_of(dout)), "lsh_embed_bwd")
        return None, dw, None, None


def embed(tokens, weight, scale=1.0, padding_idx=None):
    """scale * weight[tokens] -> [*tokens.shape, D].  tokens: int64 or int32 on the device; weight [V, D].
    Rows of padding_idx, and of ids outside the table, are zero and leave no gradient."""
    weight = _tensor(weight, "weight")
    if weight.dim() != 2 or weight.shape[1] < 1:
        raise ValueError("weight must be a [V, D] tensor")
    tokens = _tensor(tokens, "tokens", weight)
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError("tokens must be int64 or int32")
    pad = -1
    if padding_idx is not None:
        pad = int(padding_idx)
        if not 0 <= pad < weight.shape[0]:
            raise ValueError(f"padding_idx={pad} must be in the table of {weight.shape[0]} rows")
    tokens, weight = tokens.to(torch.int64).contiguous(), weight.contiguous()
    fn = EmbedFn.apply if _wants_grad(weight) else _embed_forward
    return fn(tokens, weight, float(scale), pad)


# ------------------------------------------------------------------------- distillation
def _distill_forward(logits, values, index, tau):
    rows, V = logits.shape
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    stats = torch.empty(2, rows, dtype=torch.float32, device=logits.device)
    lib = _n.lib()
    nbytes = lib.lsh_distill_workspace(rows, V)
    ws = _n.workspace(nbytes, logits.device) if nbytes else None
    with _n.on_device(logits):
        _n.check(lib.lsh_distill_fwd(
            _n.DTYPES[logits.dtype], _n.ptr(logits), logits.stride(0), _n.DTYPES[values.dtype], _n.ptr(values),
            _n.ptr(index), _n.ptr(loss), _n.ptr(stats), rows, V, values.shape[1], tau, _n.ptr(ws), nbytes,
            _n.stream_of(logits)), "lsh_distill_fwd")
    return loss, stats


class DistillFn(torch.autograd.Function):
    """distill_topk with the gradient of the student's logits."""

    @staticmethod
    def forward(ctx, logits, values, index, tau):
        loss, stats = _distill_forward(logits, values, index, tau)
        ctx.save_for_backward(logits, values, index, stats)
        ctx.tau = tau
        return loss

    @staticmethod
    def backward(ctx, g):
        logits, values, index, stats = ctx.saved_tensors
        rows, V = logits.shape
        dz = torch.empty(rows, V, dtype=logits.dtype, device=logits.device)
        with _n.on_device(logits):
            _n.check(_n.lib().lsh_distill_bwd(
                _n.DTYPES[logits.dtype], _n.ptr(logits), logits.stride(0), _n.DTYPES[values.dtype], _n.ptr(values), _n.ptr(index),
                _n.ptr(stats), _n.ptr(g), g.stride(0), _n.ptr(dz), rows, V, values.shape[1], ctx.tau,
                _n.stream_of(logits)), "lsh_distill_bwd")
        return dz, None, None, None


def distill_topk(logits, top_values, top_index, temperature=1.0):
    """Distillation from a teacher's top logits -> the loss of each row, fp32 [*rows]:

        p = softmax(top_values / tau) over the row's entries,  q = softmax(logits / tau)
        loss = tau^2 * sum_k p_k (log p_k - log q[top_index_k])

    logits [*rows, V]; top_values (any float type) and top_index (int64) [*rows, K], K up to 4096.
    An index outside the vocabulary is no entry (-1 pads short lists); a row without entries has loss 0
    and gradient 0; entries that name one id add up.  Only the logits get a gradient."""
    logits = _tensor(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [*rows, V]")
    values, index = _tensor(top_values, "top_values", logits), _tensor(top_index, "top_index", logits)
    if values.shape != index.shape or values.dim() != logits.dim() or values.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"top_values and top_index must be [*rows, K] with the rows of logits "
                         f"{tuple(logits.shape[:-1])}")
    if values.shape[-1] > MAX_K:
        raise ValueError(f"{values.shape[-1]} teacher logits a row: up to {MAX_K} are supported")
    if index.dtype != torch.int64:
        raise ValueError("top_index must be int64")
    if not values.is_floating_point():
        raise ValueError("top_values must be of a float type")
    tau = float(temperature)
    if not 0.0 < tau < float("inf"):
        raise ValueError(f"temperature={tau} must be positive and finite")
    lead, K = logits.shape[:-1], values.shape[-1]
    z = logits.reshape(-1, logits.shape[-1])
    if z.stride(1) != 1 and z.shape[1] > 1:
        z = z.contiguous()
    rows = z.shape[0]
    values = values.detach()
    if values.dtype != logits.dtype:
        values = values.to(torch.float32)
    values = values.reshape(rows, K).contiguous()
    index = index.reshape(rows, K).contiguous()
    loss = DistillFn.apply(z, values, index, tau) if _wants_grad(z) else _distill_forward(z, values, index, tau)[0]
    return loss.reshape(lead)
