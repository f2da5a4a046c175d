"""CPU: the language-model operators' C entry points check their arguments before any launch, the Python
entry points refuse host tensors, and the model's parameters are what they are documented to be."""
import ctypes

import pytest
import torch

ARG, SHAPE, WS = -1, -2, -4
P = 256  # an address that is never read: the checks fail first


def _attn(**kw):
    from lifscan import _native as n
    a = n.LinAttn(dtype=1, Dk=64, Dv=64, q_heads=4, k_heads=4, v_heads=4, T=64, B=2, H=4, q=P, k=P, v=P, beta=P, o=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_linattn_checks():
    from lifscan import _native as n
    L = n.lib()
    fwd = lambda **kw: L.lsh_linattn_fwd(_attn(**kw), None, 0, None)  # noqa: E731
    assert fwd(dtype=3) == ARG and fwd(q=None) == ARG and fwd(beta=None) == ARG and fwd(o=None) == ARG
    assert fwd(Dk=0) == SHAPE and fwd(Dv=257) == SHAPE and fwd(T=-1) == SHAPE and fwd(k_heads=3) == SHAPE
    assert fwd(B=0) == 0 and fwd(H=0) == 0
    assert L.lsh_linattn_fwd(None, None, 0, None) == ARG
    long = dict(T=8192, B=1)
    need = L.lsh_linattn_workspace(_attn(**long))
    assert need > 0 and need % (4 * 64 * 64 * 4) == 0 and L.lsh_linattn_workspace(_attn()) % 4 == 0
    assert fwd(**long) == WS and L.lsh_linattn_fwd(_attn(**long), P, need - 1, None) == WS
    bwd = lambda a, starts, ws, nb, d=P: L.lsh_linattn_bwd(a, starts, d, 1, 1, 1, None, P, P, P, None, ws, nb, None)  # noqa: E731
    nb = L.lsh_linattn_bwd_workspace(_attn(**long))
    assert nb >= need and bwd(_attn(**long), None, P, nb) == WS and bwd(_attn(**long), P, P, nb - 1) == WS
    assert bwd(_attn(**long), P, P, nb, None) == ARG
    shared = L.lsh_linattn_bwd_workspace(_attn(k_heads=1, v_heads=2, **long))
    assert shared - nb == 2 * 8192 * 4 * 64 * 4  # fp32 gradients of every head for k and v
    assert L.lsh_linattn_step(_attn(T=2), P, None) == SHAPE and L.lsh_linattn_step(_attn(T=1), None, None) == ARG


def test_row_operators_check():
    from lifscan import _native as n
    L = n.lib()
    norm = lambda **kw: n.BlockNorm(**{**dict(x_dtype=0, dtype=1, act=1, D=64, rows=8, x=P, y=P, gate=P, w_post=P,  # noqa: E731
                                              w_pre=P, eps=1e-6), **kw})
    fwd = lambda **kw: L.lsh_block_norm_fwd(ctypes.byref(norm(**kw)), P, P, None)  # noqa: E731
    assert fwd(x_dtype=2) == ARG and fwd(act=3) == ARG and fwd(gate=None) == ARG and fwd(eps=-1.0) == ARG
    assert fwd(D=0) == SHAPE and fwd(D=16385) == SHAPE and fwd(rows=-1) == SHAPE and fwd(rows=0) == 0
    assert fwd(eps=float("nan")) == ARG
    need = L.lsh_block_norm_bwd_workspace(ctypes.byref(norm()))
    assert need == 8 * 3 * 64 * 4
    assert L.lsh_block_norm_bwd(ctypes.byref(norm()), P, P, P, P, P, P, P, P, P, need - 1, None) == WS
    assert L.lsh_embed_fwd(1, None, P, P, 4, 8, 8, -1, 1.0, None) == ARG
    assert L.lsh_embed_fwd(1, P, P, P, 4, 8, 0, -1, 1.0, None) == SHAPE
    nb = L.lsh_embed_bwd_workspace(100, 1000)
    assert nb >= (2 * 1000 + 100) * 4
    assert L.lsh_embed_bwd(1, P, P, P, 100, 1000, 8, -1, 1.0, P, nb - 1, None) == WS
    assert L.lsh_embed_bwd(9, P, P, P, 100, 1000, 8, -1, 1.0, P, nb, None) == ARG
    assert L.lsh_embed_bwd(1, P, P, P, 100, 0, 8, -1, 1.0, None, 0, None) == 0
    ds = lambda dtype=1, vd=0, rows=4, V=100, K=5, tau=1.0, z=P: L.lsh_distill_fwd(  # noqa: E731
        dtype, z, V, vd, P, P, P, P, rows, V, K, tau, None, 0, None)
    assert ds(vd=2) == ARG and ds(tau=0.0) == ARG and ds(tau=float("inf")) == ARG and ds(z=None) == ARG
    assert ds(V=0) == SHAPE and ds(K=4097) == SHAPE and ds(rows=0) == 0
    assert L.lsh_distill_workspace(2, 100000) > 0 and ds(rows=2, V=100000) == WS
    assert L.lsh_distill_workspace(4096, 32000) == 0


def test_host_tensors_are_refused():
    from lifscan import hip_linattn as LA
    from lifscan import hip_lm as LM
    x, w, q = torch.zeros(4, 8), torch.ones(8), torch.zeros(4, 1, 2, 8)
    for f in (lambda: LA.lin_attn(q, q, q, 0.9), lambda: LA.lin_attn_step(q[0], q[0], q[0], 0.9, torch.zeros(1, 2, 8, 8)),
              lambda: LM.block_norm(x, x, w, w), lambda: LM.embed(torch.zeros(3, dtype=torch.int64), x),
              lambda: LM.distill_topk(x, x[:, :2], torch.zeros(4, 2, dtype=torch.int64)),
              lambda: LM.block_norm(x, x, w, w, act="relu")):
        with pytest.raises(ValueError):
            f()


def test_model_parameters():
    from lifscan.spikelm import SpikeLM
    m = SpikeLM(50, D=32, layers=2, heads=2, dk=8, dv=16, neurons=24)
    names = set(dict(m.named_parameters()))
    assert "table" in names and "blocks.1.qkv.weight" in names and "blocks.0.mix_scale" in names
    assert m.blocks[0].qkv.weight.shape == (2 * (8 + 8 + 16), 32)
    S, u = m.state(3)[0]
    assert S.shape == (3, 2, 8, 16) and u.shape == (72,)
    d = m.blocks[0].decay
    assert bool((d > 0).all()) and bool((d < 1).all()) and "blocks.0.decay" in dict(m.named_buffers())


def test_more_threads_than_a_grid_holds_are_refused():
    """A grid has fewer than 2^32 threads along an axis: what would need more is refused before the launch."""
    from lifscan import _native as n
    L = n.lib()
    assert L.lsh_linattn_step(_attn(T=1, B=2 ** 22), P, None) == SHAPE
    assert L.lsh_linattn_fwd(_attn(T=1, B=2 ** 22), None, 0, None) == SHAPE
    assert L.lsh_linattn_fwd(_attn(T=1, B=2 ** 21, Dv=128), None, 0, None) == SHAPE  # 512 threads a state
    norm = n.BlockNorm(x_dtype=0, dtype=1, act=1, D=2048, rows=2 ** 24, x=P, y=P, gate=P, w_post=P, w_pre=P, eps=1e-6)
    assert L.lsh_block_norm_fwd(ctypes.byref(norm), P, P, None) == SHAPE
    assert L.lsh_embed_fwd(1, P, P, P, 2 ** 26, 8, 512, -1, 1.0, None) == SHAPE
    assert L.lsh_distill_fwd(1, P, 8, 0, P, P, P, P, 2 ** 24, 8, 1, 1.0, None, 0, None) == SHAPE
    assert L.lsh_distill_bwd(1, P, 8, 0, P, P, P, P, 1, P, 2 ** 24, 8, 1, 1.0, None) == SHAPE


def test_linattn_without_rows_still_needs_decays():
    """The walk reads its head's decay before it looks for rows."""
    from lifscan import _native as n
    L = n.lib()
    none = dict(T=0, q=None, k=None, v=None, beta=None)
    assert L.lsh_linattn_fwd(_attn(**none), None, 0, None) == ARG
    assert L.lsh_linattn_bwd(_attn(**none), None, None, 1, 1, 1, None, None, None, None, None, None, 0, None) == ARG
    assert L.lsh_linattn_fwd(_attn(**none, B=0), None, 0, None) == 0
