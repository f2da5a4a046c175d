"""GPU: linear attention with a decay for each head (lifscan.hip_linattn) against the recurrence
S_t = beta*S_{t-1} + k_t v_t^T, o_t = scale * q_t^T S_t token by token in 64 bits, and its gradients
against the adjoint recurrence in 64 bits and against differences.

Tolerances.  Every result is a sum of products whose absolute values sum to M (the same recurrence
over absolute values).  With unit roundoff u of the type (2^-8, 2^-11, 2^-24), a 16-bit type rounds a
score or a state to its type once on the way of each product and the result once: 2u*M + u*|o|, plus
fp32 sums, below (T + D + 64)*2^-24*M for any order.  In the norm the roundings are independent and
average to less than u/sqrt(3) each, so ||error|| <= u*||result|| for 16 bits (two roundings and the
fp32 part); fp32 is held to 4e-6 (some 64 roundings of independent sign).  States are fp32 in every
type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NORM = {torch.float32: 4e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _inputs(dtype, T, B, heads, H, Dk, Dv, dev, seed=0, s0=True):
    g = torch.Generator().manual_seed(seed + T)
    hq, hk, hv = heads
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = (mk(T, B, h, d).to(dtype) for h, d in ((hq, Dk), (hk, Dk), (hv, Dv)))
    beta = 1 - torch.exp2(-torch.linspace(2, 9, H)) * (0.9 + 0.1 * torch.rand(H, generator=g))
    S = 2 * mk(B, H, Dk, Dv) if s0 else None
    do, ds = mk(T, B, H, Dv).to(dtype), 0.5 * mk(B, H, Dk, Dv)
    return [t.to(dev) if t is not None else None for t in (q, k, v, beta, S, do, ds)]


def reference(q, k, v, beta, s0, scale, do=None, ds=None):
    """The definitions in 64 bits on the CPU -> (o, s_end[, dq, dk, dv, ds0])."""
    q, k, v, beta = (t.detach().double().cpu() for t in (q, k, v, beta))
    H = beta.numel()
    share = [H // t.shape[2] for t in (q, k, v)]
    q, k, v = (t.repeat_interleave(r, 2) for t, r in zip((q, k, v), share))
    T, B, _, Dk = q.shape
    Dv = v.shape[-1]
    b = beta[:, None, None]
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64) if s0 is None else s0.detach().double().cpu()
    o = torch.zeros(T, B, H, Dv, dtype=torch.float64)
    back = do is not None or ds is not None
    if back:
        do = torch.zeros_like(o) if do is None else do.double().cpu()
        E = torch.zeros_like(S) if ds is None else ds.double().cpu()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T):
        S = b * S + k[t][..., :, None] * v[t][..., None, :]
        o[t] = scale * (q[t][..., None, :] @ S)[..., 0, :]
        if back:
            dq[t] = scale * (S @ do[t][..., :, None])[..., 0]
    if not back:
        return o, S
    for t in range(T - 1, -1, -1):
        G = E + scale * q[t][..., :, None] * do[t][..., None, :]
        dk[t] = (G @ v[t][..., :, None])[..., 0]
        dv[t] = (k[t][..., None, :] @ G)[..., 0, :]
        E = b * G
    dq, dk, dv = (d.unflatten(2, (-1, r)).sum(3) for d, r in zip((dq, dk, dv), share))
    return o, S, dq, dk, dv, E


def check(got, want, most, dtype, T, D):
    """got against want; most: the sum of the absolute values of want's products."""
    u = U[got.dtype]
    assert got.dtype in (dtype, torch.float32) and tuple(got.shape) == tuple(want.shape)
    err = (got.detach().double().cpu() - want).abs()
    bound = u * want.abs() + ((2 * u if u > 1e-6 else 0.0) + (T + D + 64) * 2.0 ** -24) * most
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())
    if want.numel() > 2000:
        assert float(err.norm()) <= NORM[got.dtype] * float(want.norm())


def _absolute(q, k, v, beta, s0, scale, *grads):
    return reference(q.abs(), k.abs(), v.abs(), beta, None if s0 is None else s0.abs(), abs(scale),
                     *(None if t is None else t.abs() for t in grads))


def run_all(q, k, v, beta, s0, scale, do, ds):
    from lifscan import hip_linattn as LA
    ins = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, v, s0)]
    o, s_end = LA.lin_attn(*ins[:3], beta, s0=ins[3], scale=scale)
    outs = [(t, g) for t, g in ((o, do), (s_end, ds)) if g is not None]
    grads = torch.autograd.grad([t for t, _ in outs], [t for t in ins if t is not None], [g for _, g in outs])
    return (o, s_end, *grads)


SHAPES = [  # T, B, (Hq, Hk, Hv), H, Dk, Dv
    (1, 1, (1, 1, 1), 1, 1, 1),
    (1, 3, (4, 4, 4), 4, 64, 64),
    (2, 2, (4, 2, 2), 4, 128, 128),
    (31, 2, (2, 2, 2), 2, 64, 128),
    (32, 1, (4, 1, 1), 4, 32, 64),
    (33, 1, (1, 1, 4), 4, 17, 40),
    (63, 2, (2, 1, 2), 2, 48, 80),
    (64, 1, (3, 3, 3), 3, 128, 64),
    (65, 2, (4, 4, 2), 4, 100, 7),
    (129, 1, (2, 2, 2), 2, 128, 128),
    (200, 1, (2, 2, 2), 2, 256, 48),
    (191, 2, (1, 1, 1), 1, 40, 256),
    (515, 1, (2, 1, 1), 2, 256, 256),
    (130, 9, (16, 16, 16), 16, 24, 16),
]


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"T{s[0]}-{s[4]}x{s[5]}")
def test_forward_and_gradients(dev, dtype, shape):
    T, B, heads, H, Dk, Dv = shape
    print(f"linattn {dtype} {shape}", flush=True)
    args = _inputs(dtype, T, B, heads, H, Dk, Dv, dev)
    scale = Dk ** -0.5
    q, k, v, beta, s0, do, ds = args
    got = run_all(q, k, v, beta, s0, scale, do, ds)
    want = reference(q, k, v, beta, s0, scale, do, ds)
    most = _absolute(q, k, v, beta, s0, scale, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, dtype, T, max(Dk, Dv))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,B,H,Dk,Dv", [(5000, 1, 1, 64, 64), (2300, 1, 2, 128, 128), (1801, 2, 2, 32, 200)])
def test_long_sequences_of_few_heads(dev, dtype, T, B, H, Dk, Dv):
    """The time axis split over workgroups and joined."""
    print(f"linattn long {dtype} {T} {B} {H} {Dk} {Dv}", flush=True)
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, B, (H,) * 3, H, Dk, Dv, dev, seed=3)
    got = run_all(q, k, v, beta, s0, 0.1, do, ds)
    want = reference(q, k, v, beta, s0, 0.1, do, ds)
    most = _absolute(q, k, v, beta, s0, 0.1, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, dtype, T, max(Dk, Dv))


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,B,H,Dk,Dv", [(1500, 1, 1, 33, 127), (701, 2, 1, 63, 7), (400, 1, 2, 129, 65),
                                         (333, 1, 1, 5, 3)])
def test_odd_widths_in_segments(dev, dtype, T, B, H, Dk, Dv):
    """Rows that begin anywhere, short first chunks, several segments, both directions."""
    print(f"linattn odd {dtype} {T} {B} {H} {Dk} {Dv}", flush=True)
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, B, (H,) * 3, H, Dk, Dv, dev, seed=7)
    got = run_all(q, k, v, beta, s0, 0.1, do, ds)
    want = reference(q, k, v, beta, s0, 0.1, do, ds)
    most = _absolute(q, k, v, beta, s0, 0.1, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, dtype, T, max(Dk, Dv))


@pytest.mark.parametrize("which", ["no_s0", "only_o", "only_state"])
def test_parts_of_the_gradient(dev, which):
    dtype, T = torch.float32, 70
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, 2, (2, 2, 2), 2, 32, 48, dev, seed=5)
    if which == "no_s0":
        s0 = None
    elif which == "only_o":
        ds = None
    else:
        do = None
    got = run_all(q, k, v, beta, s0, 0.2, do, ds)
    want = reference(q, k, v, beta, s0, 0.2, do, ds)
    most = _absolute(q, k, v, beta, s0, 0.2, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, dtype, T, 48)


@pytest.mark.parametrize("beta", [0.0, 1.0, 1e-30, 0.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_decays_at_the_ends(dev, beta, dtype):
    """A decay of 0 keeps the newest token only, 1 forgets nothing, a tiny one underflows; also as one
    number for all heads."""
    from lifscan import hip_linattn as LA
    T, H = 100, 2
    q, k, v, _, s0, do, ds = _inputs(dtype, T, 1, (H,) * 3, H, 64, 64, dev, seed=9)
    b = torch.full((H,), beta, device=dev)
    got = run_all(q, k, v, b, s0, 0.3, do, ds)
    want = reference(q, k, v, b, s0, 0.3, do, ds)
    most = _absolute(q, k, v, b, s0, 0.3, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, dtype, T, 64)
    o, s_end = LA.lin_attn(q, k, v, beta, s0=s0, scale=0.3)
    assert torch.equal(o, got[0].detach()) and torch.equal(s_end, got[1].detach())


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["batch_major", "one_projection", "shared_by_stride", "odd_offset", "last_axis"])
def test_layouts(dev, dtype, layout):
    """Strides other than the contiguous ones give the contiguous operands' bits."""
    from lifscan import hip_linattn as LA
    T, B, H, D = 77, 2, 2, 64
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, B, (H,) * 3, H, D, D, dev, seed=11)
    if layout == "shared_by_stride":
        q, k, v = (t[:, :, :1].contiguous().expand(T, B, H, D) for t in (q, k, v))
    plain = [t.contiguous() for t in (q, k, v)]
    if layout == "batch_major":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in plain)
    elif layout == "one_projection":
        q, k, v = torch.stack(plain, 2).unbind(2)
    elif layout == "odd_offset":
        q, k, v = (torch.cat([t.flatten()[:3], t.flatten()])[3:].view(t.shape) for t in plain)
    elif layout == "last_axis":
        q, k, v = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in plain)
    got = run_all(q, k, v, beta, s0, 0.125, do, ds)
    want = run_all(*plain, beta, s0, 0.125, do, ds)
    # operands that are read element by element take the same sums: the same bits
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    o, s_end = LA.lin_attn(q, k, v, beta, s0=s0, scale=0.125)
    assert torch.equal(o, want[0]) and torch.equal(s_end, want[1])


def test_training_copies_an_operand_once(dev):
    """Operands whose last axis is not contiguous are laid out once a call, and their gradients reach the tensors that
    were given."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Copies(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.n += func.overloadpacket in (torch.ops.aten.clone, torch.ops.aten.copy_)
            return func(*args, **(kwargs or {}))

    from lifscan import hip_linattn as LA
    q, k, v, beta, s0, do, ds = _inputs(torch.float32, 40, 3, (4, 2, 4), 4, 32, 16, dev, seed=37)
    ins = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o, s = LA.lin_attn(*ins, beta, s0=s0, scale=0.2)
    want = torch.autograd.grad((o, s), ins, (do, ds))
    late = [t.transpose(0, 3).contiguous().transpose(0, 3).requires_grad_(True) for t in (q, k, v)]
    for train in (True, False):
        with torch.set_grad_enabled(train), Copies() as seen:
            o1, s1 = LA.lin_attn(*late, beta, s0=s0, scale=0.2)
        assert seen.n == 3, (train, seen.n)
        assert torch.equal(o1, o) and torch.equal(s1, s)
        if train:
            for a, b in zip(torch.autograd.grad((o1, s1), late, (do, ds)), want):
                assert torch.equal(a, b)


def test_offsets_beyond_32_bits(dev):
    """Rows more than 2^31 elements apart."""
    from lifscan import hip_linattn as LA
    T, H, D = 3, 1, 64
    q, k, v, beta, s0, _, _ = _inputs(torch.bfloat16, T, 1, (1, 1, 1), H, D, D, dev, seed=13)
    step = 2 ** 31 - 64  # row 2 starts past 2^32 - 128
    far = torch.empty(2 * step + D, dtype=torch.bfloat16, device=dev)
    wide = far.as_strided((T, 1, H, D), (step, D, D, 1))
    wide.copy_(v)
    o, s = LA.lin_attn(q, k, wide, beta, s0=s0)
    o2, s2 = LA.lin_attn(q, k, v, beta, s0=s0)
    assert torch.equal(o, o2) and torch.equal(s, s2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_against_differences(dev, dtype):
    """The loss <o, do> + <s_end, ds> is linear in each operand, so a whole step along one operand
    changes it by <gradient, step> exactly; in fp32 (64-bit sums of the outputs) up to the outputs'
    own rounding, in bf16 up to the outputs' and the gradient's roundings, of independent signs."""
    from lifscan import hip_linattn as LA
    T, H, D = 90, 2, 64
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, 2, (H,) * 3, H, D, D, dev, seed=17)
    grads = run_all(q, k, v, beta, s0, 0.125, do, ds)[2:]
    ops = [q, k, v, s0]

    def loss(ops):
        o, s = LA.lin_attn(*ops[:3], beta, s0=ops[3], scale=0.125)
        return o, s, (o.double() * do.double()).sum() + (s.double() * ds.double()).sum()

    o, s, base = loss(ops)
    for i, gr in enumerate(grads):
        d = torch.randn(ops[i].shape, generator=torch.Generator().manual_seed(i)).to(dev, ops[i].dtype)
        moved = list(ops)
        moved[i] = (ops[i].double() + d.double()).to(ops[i].dtype)
        d = moved[i].double() - ops[i].double()
        o2, s2, after = loss(moved)
        # independent roundings: sqrt of the sum of squares, eight standard deviations
        u = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -8}[dtype]
        tol = 8 * u * (sum(float((a.double() * do.double()).norm()) ** 2 for a in (o, o2)) +
                       float((gr.double() * d).norm()) ** 2) ** 0.5
        tol += 8 * 2.0 ** -20 * sum(float((a.double() * ds.double()).norm()) for a in (s, s2))
        assert abs(float(after - base) - float((gr.double() * d).sum())) <= tol


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,heads,H,Dk,Dv", [(1, (8, 8, 8), 8, 64, 64), (3, (4, 2, 1), 4, 128, 128),
                                             (2, (1, 1, 1), 1, 1, 1), (5, (2, 2, 2), 2, 33, 70),
                                             (2, (3, 3, 3), 3, 256, 256), (1, (2, 1, 2), 2, 15, 130)])
def test_single_tokens_follow_the_recurrence(dev, dtype, B, heads, H, Dk, Dv):
    from lifscan import hip_linattn as LA
    T = 4
    q, k, v, beta, s0, _, _ = _inputs(dtype, T, B, heads, H, Dk, Dv, dev, seed=19)
    want, s_want = reference(q, k, v, beta, s0, 0.2)
    most, s_most = _absolute(q, k, v, beta, s0, 0.2)
    state = s0.clone()
    o = torch.stack([LA.lin_attn_step(q[t], k[t], v[t], beta, state, scale=0.2) for t in range(T)])
    check(o, want, most, dtype, T, max(Dk, Dv))
    check(state, s_want, s_most, dtype, T, max(Dk, Dv))


def test_prompt_then_tokens(dev):
    """A prompt in one call and its continuation token by token: the states of the whole sequence."""
    from lifscan import hip_linattn as LA
    q, k, v, beta, _, _, _ = _inputs(torch.float32, 100, 2, (2, 2, 2), 2, 64, 96, dev, seed=23)
    o, s = LA.lin_attn(q, k, v, beta, scale=0.1)
    a, state = LA.lin_attn(q[:97], k[:97], v[:97], beta, scale=0.1)
    b = [LA.lin_attn_step(q[t], k[t], v[t], beta, state, scale=0.1) for t in range(97, 100)]
    most, s_most = _absolute(q, k, v, beta, None, 0.1)
    tol = 2 * (100 + 96 + 64) * 2.0 ** -24
    assert bool(((torch.cat([a, torch.stack(b)]) - o).abs().cpu().double() <= tol * most).all())
    assert bool(((state - s).abs().cpu().double() <= tol * s_most).all())


def test_steps_whose_operands_share_memory_with_the_state(dev):
    """Queries, keys, values and decays are those from before the call, whichever part of the state they are views of."""
    from lifscan import hip_linattn as LA
    B, H, Dk, Dv = 3, 4, 64, 64
    q, k, v, beta, start, _, _ = _inputs(torch.float32, 1, B, (H, H, H), H, Dk, Dv, dev, seed=41)
    forms = {
        "rows": lambda s: s[:, :, 5], "columns": lambda s: s[..., 7], "one row": lambda s: s[1, 2, 3].expand(B, H, 64),
        "one head": lambda s: s[:, :1, 63], "one value": lambda s: s[2, 3, 63, 63].expand(B, H, 64),
        "a shift": lambda s: s.view(-1)[3:3 + B * H * 64].view(B, H, 64),
    }
    for name, of in forms.items():
        for which in range(4):
            def step(s, views):
                ops = [q[0], k[0], v[0]]
                if which == 3:
                    return LA.lin_attn_step(*ops, views[0, :1, 0].expand(H) if name == "one head" else views[0, :, 0], s, scale=0.3)
                ops[which] = views
                return LA.lin_attn_step(*ops, beta, s, scale=0.3)
            a, b = start.abs(), start.abs()  # decays are not negative
            o = step(a, of(a).clone())
            o1 = step(b, of(b))
            assert torch.equal(o, o1) and torch.equal(a, b), (name, which)


def test_no_tokens_and_no_batch(dev):
    from lifscan import hip_linattn as LA
    q, k, v, beta, s0, _, _ = _inputs(torch.float32, 0, 2, (2, 2, 2), 2, 8, 8, dev)
    o, s = LA.lin_attn(q, k, v, beta, s0=s0)
    assert o.shape == (0, 2, 2, 8) and torch.equal(s, s0)
    o, s = LA.lin_attn(q, k, v, beta)
    assert bool((s == 0).all())
    got = run_all(q, k, v, beta, s0, 1.0, o, torch.ones_like(s0))
    assert bool((got[5] == 1).all()) and got[2].shape == q.shape
    o, s = LA.lin_attn(q.new_zeros(3, 0, 2, 8), k.new_zeros(3, 0, 2, 8), v.new_zeros(3, 0, 2, 8), beta)
    assert o.shape == (3, 0, 2, 8) and s.shape == (0, 2, 8, 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_same_bits_on_every_run_and_stream(dev, dtype):
    q, k, v, beta, s0, do, ds = _inputs(dtype, 700, 1, (4, 2, 2), 4, 64, 64, dev, seed=29)
    first = run_all(q, k, v, beta, s0, 0.1, do, ds)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run_all(q, k, v, beta, s0, 0.1, do, ds)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_graph_replays(dev):
    """A prompt and a token captured in a HIP graph, replayed three times with eager work between."""
    from lifscan import hip_linattn as LA
    q, k, v, beta, s0, _, _ = _inputs(torch.bfloat16, 1000, 1, (2, 2, 2), 2, 64, 64, dev, seed=31)
    state = s0.clone()

    def work():
        o, s = LA.lin_attn(q, k, v, beta, s0=state, scale=0.1)
        state.copy_(s)
        return o, LA.lin_attn_step(q[0], k[0], v[0], beta, state, scale=0.1)

    want = []
    for _ in range(4):
        want.append([t.clone() for t in work()] + [state.clone()])
    state.copy_(s0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for r in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([*outs, state], want[r]):
            assert torch.equal(a, b), r
        LA.lin_attn(q, k, v, beta)  # eager work between the replays
        torch.cuda.synchronize()


def test_values_that_are_not_finite_stay_in_their_rows(dev):
    """An infinite q row is its own row's matter; a NaN value reaches the rows after it, not those
    before it."""
    from lifscan import hip_linattn as LA
    for dtype in U:
        q, k, v, beta, _, _, _ = _inputs(dtype, 100, 1, (1, 1, 1), 1, 64, 64, dev, seed=37)
        q[10, 0, 0, 3] = float("inf")
        v[70, 0, 0, 5] = float("nan")
        o, s = LA.lin_attn(q, k, v, beta, scale=0.1)
        bad = ~torch.isfinite(o[:, 0, 0])
        assert bool(bad[10].all()) and not bool(bad[:10].any()) and not bool(bad[11:70].any())
        assert bool(bad[70:, 5].all()) and int(bad[70:].sum()) == 30
        assert int((~torch.isfinite(s)).sum()) == 64


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("T,Dk,Dv", [(5, 64, 64), (300, 64, 128), (97, 33, 20)])
def test_the_error_is_that_of_one_rounding(dev, dtype, T, Dk, Dv):
    """Scores and states enter the products with 16 bits and more (2^-16 of each term, the result is rounded to
    2^-9 or 2^-12 of itself), so the error's norm is that of rounding the exact results, within a tenth."""
    args = _inputs(dtype, T, 2, (3, 3, 3), 3, Dk, Dv, dev, seed=51)
    q, k, v, beta, s0, do, ds = args
    got = run_all(q, k, v, beta, s0, Dk ** -0.5, do, ds)
    want = reference(q, k, v, beta, s0, Dk ** -0.5, do, ds)
    for x, w in zip(got, want):
        if x.dtype == dtype:
            once = float((w.to(dtype).double() - w).norm())
            err = float((x.detach().double().cpu() - w).norm())
            assert err <= 1.1 * once, (err, once)


@pytest.mark.parametrize("qk,vv", [(1e4, 1.0), (1e-3, 1.0), (1.0, 3000.0), (1.0, 2.0 ** -12)])
def test_fp16_beyond_its_range_on_the_way(dev, qk, vv):
    """Scores and states that fp16 cannot hold, or only among its smallest numbers, between operands and
    results that it can: products of q and k of that size, values of that size."""
    dtype, T, H, D = torch.float16, 150, 2, 64
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, 1, (H,) * 3, H, D, D, dev, seed=41)
    q, k, v, s0 = q * qk ** 0.5, k * qk ** 0.5, v * vv, s0 * qk ** 0.5 * vv
    do, ds, scale = do / max(vv, 1.0), ds / (qk ** 0.5 * vv), qk ** -0.5 / 16
    got = run_all(q, k, v, beta, s0, scale, do, ds)
    want = reference(q, k, v, beta, s0, scale, do, ds)
    most = _absolute(q, k, v, beta, s0, scale, do, ds)
    for g, w, m in zip(got, want, most):
        assert g.dtype != dtype or float(w.abs().max()) < 65504
        small = 2.0 ** -24 if g.dtype == dtype else 0.0  # fp16's smallest step
        err = (g.detach().double().cpu() - w).abs()
        assert bool((err <= U[g.dtype] * w.abs() + (2 * U[dtype] + (T + D + 64) * 2.0 ** -24) * m + small).all())


def _hooked(f, unpack):
    with torch.autograd.graph.saved_tensors_hooks(lambda x: (x.device, x.cpu()), unpack):
        outs, ins, grads = f()
    return torch.autograd.grad(outs, ins, grads)


def test_saved_tensors_that_come_back_changed(dev):
    """Saved operands that went through host memory give the same gradients; ones that come back in
    another type are refused, and so are second derivatives."""
    from lifscan import hip_linattn as LA
    from lifscan import hip_lm as LM
    q, k, v, beta, s0, do, ds = _inputs(torch.bfloat16, 600, 1, (2, 1, 2), 2, 32, 64, dev, seed=43)
    W, tok = torch.randn(50, 16, device=dev), torch.arange(40, device=dev) % 50
    x, w = torch.randn(6, 40, device=dev), torch.ones(40, device=dev)
    z, idx = torch.randn(5, 70, device=dev), torch.arange(15, device=dev).view(5, 3)

    def attn():
        ins = [t.detach().clone().requires_grad_(True) for t in (q, k, v, s0)]
        return LA.lin_attn(*ins[:3], beta, s0=ins[3]), ins, (do, ds)

    def norm():
        ins = [t.detach().clone().requires_grad_(True) for t in (x, x, w, w)]
        return LM.block_norm(ins[0], ins[1], ins[2], ins[3], gate=ins[1], res_scale=ins[2]), ins, (x, x)

    def lookup():
        a = W.clone().requires_grad_(True)
        out = LM.embed(tok, a)
        return out, [a], out.detach()

    def loss():
        a = z.clone().requires_grad_(True)
        return LM.distill_topk(a, z[:, :3], idx), [a], torch.ones(5, device=dev)

    for f in (attn, norm, lookup, loss):
        outs, ins, grads = f()
        want = torch.autograd.grad(outs, ins, grads)
        for a, b in zip(_hooked(f, lambda p: p[1].to(p[0])), want):
            assert torch.equal(a, b)
        with pytest.raises(ValueError):
            _hooked(f, lambda p: p[1].to(p[0]).double())
        with pytest.raises(ValueError):
            _hooked(f, lambda p: p[1])
        outs, ins, grads = f()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(outs, ins, grads, create_graph=True)


def test_refusals(dev):
    from lifscan import hip_linattn as LA
    q = torch.randn(4, 2, 2, 8, device=dev)
    b = torch.full((2,), 0.9, device=dev)
    s = torch.zeros(2, 2, 8, 8, device=dev)
    bad = [
        lambda: LA.lin_attn(q.cpu(), q.cpu(), q.cpu(), b),
        lambda: LA.lin_attn(q.double(), q.double(), q.double(), b),
        lambda: LA.lin_attn(q, q.half(), q, b),
        lambda: LA.lin_attn(q[0], q[0], q[0], b),
        lambda: LA.lin_attn(q, q[:3], q, b),
        lambda: LA.lin_attn(q, q[..., :4], q, b),
        lambda: LA.lin_attn(q, q, q, torch.full((3,), 0.9, device=dev)),
        lambda: LA.lin_attn(q, q, q, b.cpu()),
        lambda: LA.lin_attn(q, q, q, -0.5),
        lambda: LA.lin_attn(q, q, q, float("nan")),
        lambda: LA.lin_attn(q, q, q, b.clone().requires_grad_(True)),
        lambda: LA.lin_attn(q, q, q, b, s0=s[:1]),
        lambda: LA.lin_attn(q, q, q, b, s0=s.half()),
        lambda: LA.lin_attn(torch.randn(4, 2, 2, 257, device=dev), torch.randn(4, 2, 2, 257, device=dev), q, b),
        lambda: LA.lin_attn_step(q, q, q, b, s),
        lambda: LA.lin_attn_step(q[0], q[0], q[0], b, s.transpose(2, 3)),
        lambda: LA.lin_attn_step(q[0], q[0], q[0], b, s.half()),
        lambda: LA.lin_attn_step(q[0].clone().requires_grad_(True), q[0], q[0], b, s),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)


def test_a_state_changed_in_place_is_noticed(dev):
    """A graph that has saved a state must not take its gradients from the state after another token."""
    from lifscan import hip_linattn as LA
    q, k, v, beta, s0, _, _ = _inputs(torch.float32, 40, 1, (2, 2, 2), 2, 16, 16, dev, seed=31)
    o, _ = LA.lin_attn(q.requires_grad_(True), k, v, beta, s0=s0)
    with torch.no_grad():
        LA.lin_attn_step(q[0], k[0], v[0], beta, s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():  # such tensors count no versions
        LA.lin_attn_step(q[0], k[0], v[0], beta, s0.clone())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("beta", [-0.5, float("nan")])
def test_what_is_no_decay_gives_nan(dev, dtype, beta):
    """A decay below zero, or NaN, on the device: its head's results are NaN, the other heads' as they are."""
    T, H = 70, 3
    q, k, v, b, s0, do, ds = _inputs(dtype, T, 2, (H,) * 3, H, 32, 48, dev, seed=37)
    want = run_all(q, k, v, b, s0, 0.3, do, ds)
    b = b.clone()
    b[1] = beta
    got = run_all(q, k, v, b, s0, 0.3, do, ds)
    for i, (x, w) in enumerate(zip(got, want)):
        heads = 1 if i in (1, 5) else 2  # states [B, H, ...], the others [T, B, H, ...]
        assert bool(x.select(heads, 1).isnan().all())
        for h in (0, 2):
            assert torch.equal(x.select(heads, h), w.select(heads, h))


@pytest.mark.parametrize("Dv", [48, 50])
@pytest.mark.parametrize("beta", [-0.5, float("nan")])
def test_what_is_no_decay_gives_nan_in_a_step(dev, beta, Dv):
    from lifscan import hip_linattn as LA
    q, k, v, b, s0, _, _ = _inputs(torch.float32, 1, 2, (3,) * 3, 3, 32, Dv, dev, seed=41)
    good, bad = s0.clone(), s0.clone()
    want = LA.lin_attn_step(q[0], k[0], v[0], b, good)
    b = b.clone()
    b[1] = beta
    got = LA.lin_attn_step(q[0], k[0], v[0], b, bad)
    assert bool(got[:, 1].isnan().all()) and bool(bad[:, 1].isnan().all())
    for h in (0, 2):
        assert torch.equal(got[:, h], want[:, h]) and torch.equal(bad[:, h], good[:, h])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("what", ["state", "scores"])
def test_cancelling_terms_keep_the_digits_of_fp32(dev, dtype, what):
    """Two terms of an output that cancel but for their last digits, from the state or from two scores: scores
    and states are fp32 numbers, so an output is off by its own rounding and a few 2^-24 of its terms (six
    products at most that are added in fp32, fp16's parts of 22 bits and more, and the factors of the decays: 16
    in all).  Sixteen bits would leave some 2^-17 of them."""
    from lifscan import hip_linattn as LA
    B, H, Dv = 3, 4, 80
    g = torch.Generator().manual_seed(61)
    beta = 1 - torch.exp2(-torch.linspace(2, 9, H))
    if what == "state":
        T, Dk = 1, 2
        q, k = torch.ones(T, B, H, Dk), torch.zeros(T, B, H, Dk)
        v = torch.randn(T, B, H, Dv, generator=g)
        s0 = 1 + torch.rand(B, H, Dk, Dv, generator=g)
        s0[:, :, 1] = -s0[:, :, 0] + 2.0 ** -12 * torch.rand(B, H, Dv, generator=g)
    else:
        T, Dk = 2, 4
        beta = torch.ones(H)
        q = 1 + torch.rand(T, B, H, Dk, generator=g)
        k = (1 + torch.rand(1, B, H, Dk, generator=g)).to(dtype).float().repeat(T, 1, 1, 1)
        k[:, ..., 3] = torch.tensor([2.0 ** -11, 2.0 ** -12])[:, None, None]
        v = torch.ones(T, B, H, Dv)
        v[1] = -1
        s0 = None
    q, k, v, beta = q.to(dtype).to(dev), k.to(dtype).to(dev), v.to(dtype).to(dev), beta.to(dev)
    s0 = None if s0 is None else s0.to(dev)
    o, _ = LA.lin_attn(q, k, v, beta, s0=s0)
    want, _ = reference(q, k, v, beta, s0, 1.0)
    most, _ = _absolute(q, k, v, beta, s0, 1.0)
    err = (o.double().cpu() - want)[-1].abs()
    bound = U[dtype] * want[-1].abs() + 16 * 2.0 ** -24 * most[-1] + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert float((want[-1].abs() / most[-1]).max()) < 2.0 ** -10
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,beta", [(1, 20.0), (2, 20.0), (5, 20.0), (3, 300.0), (1, 1e30), (27, 20.0), (64, 3.0)])
def test_decays_that_grow(dev, dtype, T, beta):
    """Any finite factor is a decay: what a chunk has no rows for must not overflow where the results do not."""
    H, D = 2, 24
    q, k, v, b, s0, do, ds = _inputs(dtype, T, 2, (H,) * 3, H, D, D, dev, seed=67)
    b = torch.tensor([beta, 0.5], device=dev)
    size = beta ** -(T - 1)  # so that 16-bit results stay in their type's range
    scale = min(max(size, 2.0 ** -100), 1.0)
    s0, ds = s0 / 2 ** 10, ds * scale
    if dtype == torch.float16:
        scale = scale / 2 ** 8 / beta if beta < 1e10 else 1e-30
        ds = ds / 2 ** 8 / beta if beta < 1e10 else ds * 1e-30
        s0 = s0 / beta
    got = run_all(q, k, v, b, s0, scale, do, ds)
    want = reference(q, k, v, b, s0, scale, do, ds)
    most = _absolute(q, k, v, b, s0, scale, do, ds)
    for x, w, m in zip(got, want, most):
        small = 2.0 ** -24 if x.dtype == torch.float16 else 0.0
        err = (x.detach().double().cpu() - w).abs()
        u = U[x.dtype]
        # a power of beta: its exponent, up to log2(beta^T) <= 128, is an fp32 number
        bound = u * w.abs() + ((2 * u if u > 1e-6 else 0.0) + (T + D + 64 + 128) * 2.0 ** -24) * m + small
        assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,Dk", [(70, 64), (330, 128)])
def test_rows_of_zeros_do_not_grow(dev, dtype, T, Dk):
    """Zeros times any power of a decay are zeros: a sequence whose first rows (for the gradients: last rows) are
    zeros, in one segment and in several."""
    from lifscan import hip_linattn as LA
    H, Dv, beta = 1, 64, 20.0
    q, k, v, _, _, do, _ = _inputs(dtype, T, 1, (H,) * 3, H, Dk, Dv, dev, seed=71, s0=False)
    b = torch.full((H,), beta, device=dev)
    late, early = v.clone(), do.clone()
    late[:-4] = 0
    early[4:] = 0
    o, s = LA.lin_attn(q, k, late, b, scale=2.0 ** -20)
    want, s_want = reference(q, k, late, b, None, 2.0 ** -20)
    most, s_most = _absolute(q, k, late, b, None, 2.0 ** -20)
    check(o, want, most, dtype, T, Dk)
    check(s, s_want, s_most, dtype, T, Dk)
    got = run_all(q, k, late * 0, b, None, 2.0 ** -20, early, None)
    want = reference(q, k, late * 0, b, None, 2.0 ** -20, early, None)
    most = _absolute(q, k, late * 0, b, None, 2.0 ** -20, early, None)
    for i in (2, 3, 4):
        check(got[i], want[i], most[i], dtype, T, Dk)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_slow_decays_of_long_sequences_do_not_drift(dev, dtype):
    """The first state after T rows without values is beta^T times it.  Bound: beta^T = 2^(T*log2 beta) with
    T*log2 beta up to 6, the logarithm off by 2^-23 of itself and its product by 2^-24 (12 * 2^-24 of the result),
    the power by 2^-23, and one rounding each for its product with the state and where the state is rescaled: below
    24 * 2^-24.  Heads enough that no row is split."""
    from lifscan import hip_linattn as LA
    T, B, D = 16384, 172, 8
    beta = torch.tensor([1 - 2.0 ** -12, 1 - 2.0 ** -14, 1 - 2.0 ** -16])
    g = torch.Generator().manual_seed(73)
    s0 = 1 + torch.rand(B, 3, D, D, generator=g)
    z = torch.zeros(T, B, 3, D, dtype=dtype, device=dev)
    _, s = LA.lin_attn(z, z, z, beta.to(dev), s0=s0.to(dev))
    want = s0.double() * beta.double()[:, None, None] ** T
    err = (s.double().cpu() - want).abs() / want
    assert float(err.max()) <= 24 * 2.0 ** -24, [float(e) / 2.0 ** -24 for e in err.amax((0, 2, 3))]


def test_step_refuses_a_decay_that_asks_for_a_gradient(dev):
    from lifscan import hip_linattn as LA
    q, s = torch.randn(2, 2, 8, device=dev), torch.zeros(2, 2, 8, 8, device=dev)
    b = torch.full((2,), 0.9, device=dev, requires_grad=True)
    with pytest.raises(ValueError, match="beta"):
        LA.lin_attn_step(q, q, q, b, s)
    assert bool((s == 0).all())
    with torch.no_grad():
        LA.lin_attn_step(q, q, q, b, s)
    assert not bool((s == 0).all())


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,H", [(100, 600), (300, 1)])
def test_infinite_values_reach_what_depends_on_them(dev, dtype, T, H):
    """An infinite value, or element of the first state: its column from its row on (the state's element alone) is
    not finite, whole and in segments, and nothing else."""
    from lifscan import hip_linattn as LA
    q, k, v, beta, s0, _, _ = _inputs(dtype, T, 1, (1, 1, 1), H, 32, 48, dev, seed=79)
    v[20, 0, 0, 5], v[T - 1, 0, 0, 11] = float("inf"), float("-inf")
    s0[0, 0, 3, 9] = float("inf")
    o, s = LA.lin_attn(q, k, v, beta, s0=s0, scale=0.1)
    want_o, want_s = torch.ones_like(o, dtype=torch.bool), torch.ones_like(s, dtype=torch.bool)
    want_o[20:, 0, :, 5] = want_o[T - 1, 0, :, 11] = want_o[:, 0, 0, 9] = False
    want_s[0, :, :, 5] = want_s[0, :, :, 11] = want_s[0, 0, 3, 9] = False
    assert torch.equal(o.isfinite(), want_o) and torch.equal(s.isfinite(), want_s)


def test_more_pairs_than_one_launch_of_the_three_walks_holds(dev):
    """What the forward takes the gradients take: 6 million (batch, head) pairs, whose three walks have too many
    threads for one launch."""
    from lifscan import hip_linattn as LA
    T, B, H = 2, 3 << 20, 2
    q, k, v, do = (torch.rand(T, B, H, 1, device=dev, generator=torch.Generator(dev).manual_seed(i)) for i in range(4))
    beta = torch.tensor([0.5, 0.25], device=dev)
    ins = [t.requires_grad_(True) for t in (q, k, v)]
    o, s = LA.lin_attn(*ins, beta)
    dq, dk, dv = torch.autograd.grad(o, ins, do)
    q, k, v = (t.detach() for t in (q, k, v))
    b = beta[:, None]
    kv = k * v
    S1 = b * kv[0] + kv[1]
    G0 = q[0] * do[0] + b * q[1] * do[1]
    for got, want in ((o[1], q[1] * S1), (s[..., 0], S1), (dq[1], S1 * do[1]), (dk[0], G0 * v[0]), (dv[0], G0 * k[0])):
        assert float((got.detach() - want).abs().max()) < 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("first", ["none", "aligned", "odd_offset"])
def test_many_states_in_segments(dev, dtype, first):
    """2^19 state elements in eight segments (fp32) and eleven, joined four elements and eight segments at a time; a
    first state that does not begin at a multiple of 16 bytes is joined one by one.  A decay of its own for each head."""
    T, B, H, Dk, Dv = 700, 2, 16, 128, 128
    print(f"linattn join {dtype} {first}", flush=True)
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, B, (H,) * 3, H, Dk, Dv, dev, seed=83)
    if first == "none":
        s0 = None
    elif first == "odd_offset":
        s0 = torch.cat([s0.flatten()[:1], s0.flatten()])[1:].view(s0.shape)
    got = run_all(q, k, v, beta, s0, 0.1, do, ds)
    want = reference(q, k, v, beta, s0, 0.1, do, ds)
    most = _absolute(q, k, v, beta, s0, 0.1, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, dtype, T, Dk)


@pytest.mark.parametrize("T,H,Dk,Dv", [(150, 2, 129, 256), (150, 1, 256, 140), (40, 2, 200, 130)])
def test_walks_of_unequal_column_blocks_in_one_launch(dev, T, H, Dk, Dv):
    """fp32 gradients whose walks have three and four (four and three) blocks of columns."""
    q, k, v, beta, s0, do, ds = _inputs(torch.float32, T, 2, (H,) * 3, H, Dk, Dv, dev, seed=89)
    got = run_all(q, k, v, beta, s0, 0.1, do, ds)
    want = reference(q, k, v, beta, s0, 0.1, do, ds)
    most = _absolute(q, k, v, beta, s0, 0.1, do, ds)
    for g, w, m in zip(got, want, most):
        check(g, w, m, torch.float32, T, 256)


@pytest.mark.parametrize("qk,vv", [(2.0 ** -10, 1.0), (1.0, 2.0 ** -20), (2.0 ** -8, 2.0 ** -18), (1e4, 1.0), (1.0, 3000.0)])
def test_fp16_states_and_scores_hold_22_bits_at_any_size(dev, qk, vv):
    """fp16 operands far below (and above) one: states, outputs and gradients that are scaled back to about one.
    An output is off by its own rounding and 2^-22 of its terms for a score's and a state's parts, a state by 2^-22
    for the decayed values' parts; both by fp32 sums.  Parts that were not scaled would leave 2^-25 of an absolute
    size to each, which at values of 2^-20 is 2^-5 of them."""
    dtype, T, H, D = torch.float16, 150, 2, 64
    q, k, v, beta, s0, do, ds = _inputs(dtype, T, 1, (H,) * 3, H, D, D, dev, seed=97)
    q, k, v, s0 = q * qk ** 0.5, k * qk ** 0.5, v * vv, s0 * (qk ** 0.5 * vv)
    scale = 2.0 ** -4 / (qk * vv)
    do, ds = do * min(vv * qk ** 0.5 * 2.0 ** 4, 1.0), ds * min(1.0 / (qk ** 0.5 * vv), 2.0 ** 8)
    got = run_all(q, k, v, beta, s0, scale, do, ds)
    want = reference(q, k, v, beta, s0, scale, do, ds)
    most = _absolute(q, k, v, beta, s0, scale, do, ds)
    for x, w, m in zip(got, want, most):
        assert x.dtype != dtype or float(w.abs().max()) < 65504
        small = 2.0 ** -25 if x.dtype == dtype else 0.0  # half of fp16's smallest step
        err = (x.detach().double().cpu() - w).abs()
        bound = U[x.dtype] * w.abs() + (2 * 2.0 ** -22 + (T + D + 64) * 2.0 ** -24) * m + small
        assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())
