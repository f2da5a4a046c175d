"""The row operators of a spiking language model on MI355X: what stands between its neurons
(``hip_lif``), its mixing layers (``hip_linattn``) and its matrix products.

  block_norm    the norm after a block, its gate and residual scale, and the norm before the next block
  embed         embedding lookup with scaling; the table's gradient sums by token
  distill_topk  the loss against a teacher's top logits
  token_logprobs  log probabilities of given tokens, the entropy, the most likely alternatives

Tensors are float32, bfloat16 or float16; sums and statistics are fp32 and every result is rounded to
its tensor's type once.  Every operator is deterministic (no floating-point atomics).  No counterpart
in the reference.  There is no fallback: every call runs the HIP kernels of liblifscan_hip.so through
the C++ operators of ``_ops_lm.cpp``, which check the arguments and raise ValueError.
"""
import torch

from . import _native as _n

GATES = {"silu": 1, "sigmoid": 2}  # LSH_GATE_*


def block_norm(x, y, w_post, w_pre, gate=None, res_scale=1.0, eps=1e-6, act="silu"):
    """The end of one block and the start of the next, rows along the last axis -> (x_new, z):

        n = y / sqrt(mean(y^2) + eps) * w_post          the block's output y, normalised
        x_new = x + res_scale * act(gate) * n           the residual stream
        z = x_new / sqrt(mean(x_new^2) + eps) * w_pre   the next block's input

    x (the residual stream) is float32 or has y's type; y and gate have one type; up to 16384 channels.
    w_post, w_pre: [D].  gate: like y, or None (no gate); act: "silu" or "sigmoid".  res_scale: a number,
    or a [D] tensor with its own gradient.  z is taken from x_new before that is rounded."""
    if act not in GATES:
        raise ValueError(f"act {act!r}: 'silu' or 'sigmoid'")
    tensor = torch.is_tensor(res_scale)
    return _n.lm_ops().block_norm(x, y, w_post, w_pre, gate, res_scale if tensor else None,
                                  0.0 if tensor else float(res_scale), eps, GATES[act])


def embed(tokens, weight, scale=1.0, padding_idx=None):
    """scale * weight[tokens] -> [*tokens.shape, D].  tokens: int64 or int32 on the device; weight [V, D].
    Rows of padding_idx, and of ids outside the table, are zero and leave no gradient.  The gradient is
    dense; a token's rows are summed in an order that depends on the tokens alone."""
    return _n.lm_ops().embed(tokens, weight, scale, padding_idx)


def distill_topk(logits, top_values, top_index, temperature=1.0):
    """Distillation from a teacher's top logits -> the loss of each row, fp32 [*rows]:

        p = softmax(top_values / tau) over the row's entries,  q = softmax(logits / tau)
        loss = tau^2 * sum_k p_k (log p_k - log q[top_index_k])

    logits [*rows, V]; top_values (any float type) and top_index (int64) [*rows, K], K up to 4096.
    An index outside the vocabulary is no entry (-1 pads short lists); a row without entries has loss 0
    and gradient 0; entries that name one id add up.  Only the logits get a gradient."""
    return _n.lm_ops().distill_topk(logits, top_values, top_index, temperature)


def token_logprobs(logits, tokens, temperature=1.0, top=0):
    """What a model says about given tokens -> (logp, entropy), fp32 [*rows]; with top = K > 0 also the most
    likely alternatives (top_logp fp32, top_index int64), [*rows, K]:

        p = softmax(logits / tau),  logp = log p[token],  entropy = -sum p log p

    logits [*rows, V], read through its row stride; tokens [*rows], int64 or int32.  A token outside the
    vocabulary is none: logp 0 without a gradient.  Alternatives come in order, equal logits by their id, NaN
    first; top up to 64 and V.  The logits get a gradient from logp and from the entropy, not from the
    alternatives.  A logit of -inf has probability 0, as has one whose probability is below the smallest normal
    fp32 number; a row of nothing else has logp -inf, entropy 0 and no gradient, and a row with NaN or +inf has
    NaN."""
    return tuple(_n.lm_ops().token_logprobs(logits, tokens, temperature, top))
