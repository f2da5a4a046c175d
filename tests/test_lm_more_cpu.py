"""CPU: the C entry points of the gated recurrence, the heads' rotation and the tokens' log probabilities check
their arguments before any launch, and the Python entry points refuse host tensors."""
import ctypes

import pytest
import torch

ARG, SHAPE, WS = -1, -2, -4
P = 256  # an address that is never read: the checks fail first


def _gated(**kw):
    from lifscan import _native as n
    a = n.Gated(dtype=1, decay=0, mix=1, T=64, B=2, D=8, x=P, gate=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_gated_checks():
    from lifscan import _native as n
    L = n.lib()
    fwd = lambda h=P, end=P, ws=None, nb=0, **kw: L.lsh_gated_fwd(_gated(**kw), h, end, None, ws, nb, None)  # noqa: E731
    assert L.lsh_gated_fwd(None, P, P, None, None, 0, None) == ARG
    assert fwd(dtype=3) == ARG and fwd(decay=2) == ARG and fwd(decay=-1) == ARG and fwd(x=None) == ARG
    assert fwd(gate=None) == ARG and fwd(h=None) == ARG and fwd(end=None) == ARG
    assert fwd(T=-1) == SHAPE and fwd(B=-1) == SHAPE and fwd(D=0) == SHAPE and fwd(B=0) == 0
    assert fwd(B=2 ** 20, D=2 ** 21) == SHAPE and fwd(T=2 ** 30, B=2 ** 10, D=2 ** 10) == SHAPE
    need = L.lsh_gated_workspace(_gated(T=4096))
    assert need > 0 and need % (2 * 2 * 8 * 4) == 0 and L.lsh_gated_workspace(_gated()) == 0
    assert fwd(T=4096) == WS and fwd(T=4096, ws=P, nb=need - 1) == WS
    assert L.lsh_gated_saved(_gated(T=129)) == 3 * 16 and L.lsh_gated_saved(_gated(T=0)) == 0
    bwd = lambda a, saved=P, dx=P, dg=P, ws=None, nb=0: L.lsh_gated_bwd(a, saved, P, 1, 1, None, dx, dg, None, ws, nb, None)  # noqa: E731
    assert bwd(_gated(), saved=None) == ARG and bwd(_gated(), dx=None) == ARG and bwd(_gated(), dg=None) == ARG
    assert bwd(_gated(T=4096)) == WS and bwd(_gated(B=0)) == 0 and bwd(_gated(dtype=7)) == ARG
    step = lambda a, s=P, h=P: L.lsh_gated_step(a, s, h, None)  # noqa: E731
    assert step(_gated()) == SHAPE and step(_gated(T=1), s=None) == ARG and step(_gated(T=1), h=None) == ARG
    assert step(_gated(T=1, B=0)) == 0


def test_gated_segments_cover_the_rows():
    """The workspace holds whole segments of whole rounds for either width of a piece, and none when the channels
    fill the chip."""
    from lifscan import _native as n
    L = n.lib()
    for T in (128, 129, 1000, 4096, 100000):
        for B, D in ((1, 1), (1, 64), (3, 257), (4, 2048), (16, 4096)):
            nb = L.lsh_gated_workspace(_gated(T=T, B=B, D=D))
            segments = nb / (2 * B * D * 4)
            assert segments == int(segments) and segments <= -(-T // 128)
    assert L.lsh_gated_workspace(_gated(T=4096, B=16, D=4096)) == 0


def _rotate(**kw):
    from lifscan import _native as n
    a = n.Rotate(dtype=1, D=64, rot=64, T=4, B=2, H=4, HK=2, q=P, k=P, positions=P, inv_freq=P, q_weight=P, k_weight=P, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_rotate_checks():
    from lifscan import _native as n
    L = n.lib()
    fwd = lambda qo=P, ko=P, **kw: L.lsh_rotate_fwd(_rotate(**kw), qo, ko, None)  # noqa: E731
    assert L.lsh_rotate_fwd(None, P, P, None) == ARG
    assert fwd(dtype=3) == ARG and fwd(q=None) == ARG and fwd(k=None) == ARG and fwd(positions=None) == ARG
    assert fwd(inv_freq=None) == ARG and fwd(q_weight=None) == ARG and fwd(k_weight=None) == ARG and fwd(eps=-1.0) == ARG
    assert fwd(eps=float("nan")) == ARG and fwd(qo=None) == ARG and fwd(ko=None) == ARG
    for kw in (dict(D=63), dict(D=0), dict(D=258), dict(rot=66), dict(rot=31), dict(rot=-2), dict(T=-1), dict(B=-1), dict(H=-1),
               dict(HK=2 ** 17), dict(T=2 ** 40, B=2), dict(T=2 ** 32)):
        assert fwd(**kw) == SHAPE, kw
    assert fwd(T=0) == 0 and fwd(B=0) == 0 and fwd(H=0, HK=0) == 0
    need = L.lsh_rotate_bwd_workspace(_rotate())
    assert need > 0 and need % (2 * 64 * 4) == 0 and L.lsh_rotate_bwd_workspace(_rotate(q_weight=None, k_weight=None)) == 0
    bwd = lambda a, gq=P, gk=P, dq=P, dk=P, ws=P, nb=need: L.lsh_rotate_bwd(  # noqa: E731
        a, gq, 1, 1, 1, gk, 1, 1, 1, dq, dk, None, None, ws, nb, None)
    assert bwd(_rotate(), gq=None) == ARG and bwd(_rotate(), gk=None) == ARG and bwd(_rotate(), dq=None) == ARG
    assert bwd(_rotate(), nb=need - 1) == WS and bwd(_rotate(), ws=None) == WS and bwd(_rotate(T=0)) == 0


def test_score_checks():
    from lifscan import _native as n
    L = n.lib()
    f = lambda dtype=1, z=P, tok=P, lp=P, en=P, tl=P, ti=P, rows=4, V=100, K=5, tau=1.0, ws=None, nb=0: L.lsh_score_fwd(  # noqa: E731
        dtype, z, V, tok, lp, en, None, tl, ti, rows, V, K, tau, ws, nb, None)
    assert f(dtype=3) == ARG and f(tau=0.0) == ARG and f(tau=float("inf")) == ARG and f(tau=float("nan")) == ARG
    assert f(tau=1e-39) == ARG  # its reciprocal is no fp32 number
    assert f(z=None) == ARG and f(tok=None) == ARG and f(lp=None) == ARG and f(en=None) == ARG and f(tl=None) == ARG and f(ti=None) == ARG
    assert f(V=0) == SHAPE and f(K=65) == SHAPE and f(K=-1) == SHAPE and f(V=4, K=5) == SHAPE and f(rows=-1) == SHAPE
    assert f(rows=2 ** 24) == SHAPE and f(rows=0) == 0
    need = L.lsh_score_workspace(2, 100000, 5)
    assert need > 0 and f(rows=2, V=100000) == WS and f(rows=2, V=100000, ws=P, nb=need - 1) == WS
    assert L.lsh_score_workspace(4096, 32000, 5) == 0
    b = lambda dtype=1, z=P, tok=P, st=P, dz=P, rows=4, V=100, tau=1.0: L.lsh_score_bwd(  # noqa: E731
        dtype, z, V, tok, st, P, 1, P, 1, dz, rows, V, tau, None)
    assert b(dtype=3) == ARG and b(z=None) == ARG and b(tok=None) == ARG and b(st=None) == ARG and b(dz=None) == ARG
    assert b(tau=-1.0) == ARG and b(V=0) == SHAPE and b(rows=0) == 0


def test_host_tensors_are_refused():
    from lifscan import hip_gated as G
    from lifscan import hip_linattn as LA
    from lifscan import hip_lm as LM
    x, q, tok = torch.zeros(4, 2, 8), torch.zeros(4, 1, 2, 8), torch.zeros(4, dtype=torch.int64)
    for f in (lambda: G.gated_scan(x, x), lambda: G.gated_scan_step(x[0], x[0], torch.zeros(2, 8)),
              lambda: G.gated_scan(x, x, decay="none"), lambda: LA.norm_rotate(q, q, tok, torch.ones(4)),
              lambda: LA.norm_rotate(q, q, tok, torch.ones(4), pairs="none"), lambda: LM.token_logprobs(x[:, 0], tok)):
        with pytest.raises(ValueError):
            f()


def test_models_with_other_mixers():
    from lifscan.spikelm import SpikeLM
    kw = dict(D=32, layers=2, heads=2, dk=8, dv=16, neurons=24)
    plain = set(dict(SpikeLM(50, **kw).named_parameters()))
    assert not any("norm" in n or "vg" in n for n in plain)
    m = SpikeLM(50, rotary=True, **kw)
    assert set(dict(m.named_parameters())) - plain == {f"blocks.{i}.{n}" for i in range(2) for n in ("q_norm", "k_norm")}
    S, u, at = m.state(3)[0]
    assert S.shape == (3, 2, 8, 16) and u.shape == (72,) and at.shape == (3,) and at.dtype == torch.int64
    want = [10000.0 ** (-2 * i / 8) for i in range(4)]
    for n in (m, SpikeLM(50, rotary=True, **kw).bfloat16()):
        f = n.blocks[1].inv_freq
        assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-15)
        assert not any("inv_freq" in k for k in n.state_dict())
    m = SpikeLM(50, mixer="gated", **kw)
    names = dict(m.named_parameters())
    assert names["blocks.0.vg.weight"].shape == (64, 32) and names["blocks.1.gate_bias"].shape == (32,) and "blocks.0.qkv.weight" not in names
    S, u = m.state(3)[1]
    assert S.shape == (3, 32) and u.shape == (72,)
    for bad in (dict(mixer="none"), dict(mixer="gated", rotary=True)):
        with pytest.raises(ValueError):
            SpikeLM(50, **kw, **bad)
