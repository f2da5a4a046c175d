"""GPU: the gated linear recurrence (lifscan.hip_gated) against the recurrence in 64 bits row by row, its
gradients against the adjoint recurrence in 64 bits and against differences.

Tolerances.  With F = 2^-24, a decay and a weight are each off by at most 8 F of themselves (a power of two
whose argument is corrected, 1 + e, a reciprocal of 1 ulp, their product), and a row adds a product and a
sum.  Products of decays over a run of rows round as often as the rows do.  So an element is off by at most
what the recurrence e_t = a_t e_{t-1} + 24 F (a_t M_{t-1} + w_t |x_t|) gives, M being the recurrence of
absolute values, plus its own rounding u*|result|.  The adjoint is the same recurrence backwards; a gradient
multiplies both, with 24 F more for its own factors.  A 16-bit gate's exponential does not correct its
argument g*log2(e): rounded once, with log2(e) off by 0.3 F, it is off by 1.3 |g| F at most, so 24 F is
(24 + 2 |g|) F there; beyond |g| = 90 the exponential itself is below the smallest normal number."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FORMS = [("sigmoid", True), ("sigmoid", False), ("log", True), ("log", False)]


def reference(x, gate, h0, starts, decay, mix, dh=None, dend=None):
    """name -> (value, bound of its error before rounding), in 64 bits on the CPU."""
    fine = x.dtype == torch.float32
    x, gate = (t.detach().double().cpu() for t in (x, gate))
    T, B, D = x.shape
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    if decay == "sigmoid":
        a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
        slope = a * rest
    else:
        low = torch.minimum(gate, torch.zeros_like(gate))
        a, rest = torch.exp(low), -torch.expm1(low)
        slope = torch.where(gate > 0, 0.0, a)
    w = rest if mix else torch.ones_like(rest)
    C = torch.full_like(gate, 24 * F) if fine else (24 + 2 * gate.abs().clamp(max=90)) * F
    keep = torch.ones(T, B, 1, dtype=torch.bool) if starts is None else (starts.cpu() == 0)[..., None]
    out, prev, M_prev, e_prev = (torch.empty_like(x) for _ in range(4))
    e_out = torch.empty_like(x)
    M, e = h.abs(), torch.zeros_like(h)
    for t in range(T):
        zero = torch.zeros_like(h)
        h, M, e = (torch.where(keep[t], s, zero) for s in (h, M, e))
        prev[t], M_prev[t], e_prev[t] = h, M, e
        e = a[t] * e + C[t] * (a[t] * M + (w[t] * x[t]).abs())
        M = a[t] * M + (w[t] * x[t]).abs()
        h = a[t] * h + w[t] * x[t]
        out[t], e_out[t] = h, e
    res = {"h": (out, e_out), "end": (h, e)}
    if dh is None and dend is None:
        return res
    dh = torch.zeros_like(x) if dh is None else dh.detach().double().cpu()
    E = torch.zeros(B, D, dtype=torch.float64) if dend is None else dend.detach().double().cpu()
    ME, eE = E.abs(), torch.zeros_like(E)
    dx, dg, bx, bg = (torch.empty_like(x) for _ in range(4))
    for t in range(T - 1, -1, -1):
        E, ME = E + dh[t], ME + dh[t].abs()
        eE = eE + F * ME
        v = x[t] if mix else torch.zeros_like(x[t])
        size = prev[t].abs() + v.abs()
        dx[t], bx[t] = w[t] * E, w[t] * (eE + C[t] * ME)
        dg[t] = slope[t] * E * (prev[t] - v)
        bg[t] = slope[t] * (eE * size + ME * e_prev[t] + C[t] * ME * size)
        E, ME, eE = a[t] * E, a[t] * ME, a[t] * eE + C[t] * a[t] * ME
        E, ME, eE = (torch.where(keep[t], s, torch.zeros_like(s)) for s in (E, ME, eE))
    return {**res, "dx": (dx, bx), "dgate": (dg, bg), "dh0": (E, eE)}


def close(got, want, name=""):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), name
    err = (got.detach().double().cpu() - value).abs()
    bound = bound + U[got.dtype] * (value.abs() + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126)
    assert bool((err <= bound).all()), (name, float((err / bound).max()))


def inputs(T, B, D, dtype, dev, decay="sigmoid", starts=False, seed=0, shift=2.0):
    g = torch.Generator().manual_seed(1000 * seed + T + 7 * D)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, gate = mk(T, B, D), mk(T, B, D) * 1.5 + shift
    if decay == "log":
        gate = -torch.exp(-gate)
    st = torch.rand(T, B, generator=g) < 0.07 if starts else None
    out = [x.to(dtype), gate.to(dtype), mk(B, D), st, mk(T, B, D).to(dtype), mk(B, D)]
    return [t.to(dev) if t is not None else None for t in out]


def run(x, gate, h0, starts, decay, mix, dh=None, dend=None):
    from lifscan import hip_gated as G
    ins = [t.detach().requires_grad_(True) if t is not None else None for t in (x, gate, h0)]
    h, end = G.gated_scan(ins[0], ins[1], ins[2], starts=starts, decay=decay, mix=mix)
    outs = [(o, d) for o, d in ((h, dh), (end, dend)) if d is not None]
    have = [t for t in ins if t is not None]
    got = {"h": h, "end": end}
    if outs:
        grads = torch.autograd.grad([o for o, _ in outs], have, [d for _, d in outs])
        got.update(zip(("dx", "dgate", "dh0"), grads))
    return got


def check(got, want):
    for k in got:
        close(got[k], want[k], k)


SHAPES = [(1, 1, 1), (1, 3, 130), (2, 2, 2), (15, 1, 64), (16, 3, 5), (17, 2, 66), (33, 1, 127), (64, 2, 128), (65, 1, 257),
          (127, 2, 34), (128, 1, 3), (129, 3, 32), (300, 2, 50), (1000, 1, 257), (1025, 3, 6)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,B,D", SHAPES)
def test_forward_and_gradients(dev, dtype, T, B, D):
    print(f"gated {T}x{B}x{D} {dtype}", flush=True)
    decay, mix = FORMS[(T + D) % 4]
    for starts in (False, True):
        x, gate, h0, st, dh, dend = inputs(T, B, D, dtype, dev, decay, starts)
        got = run(x, gate, h0, st, decay, mix, dh, dend)
        assert got["h"].dtype == got["dx"].dtype == got["dgate"].dtype == dtype
        assert got["end"].dtype == got["dh0"].dtype == torch.float32
        check(got, reference(x, gate, h0, st, decay, mix, dh, dend))


@pytest.mark.parametrize("decay,mix", FORMS)
@pytest.mark.parametrize("starts", [False, True])
def test_every_form(dev, decay, mix, starts):
    x, gate, h0, st, dh, dend = inputs(200, 2, 48, torch.float32, dev, decay, starts, seed=1)
    check(run(x, gate, h0, st, decay, mix, dh, dend), reference(x, gate, h0, st, decay, mix, dh, dend))


# few channels: many segments; many: one; between: segments of unequal length
@pytest.mark.parametrize("T,B,D", [(9000, 1, 2), (5001, 2, 33), (2100, 5, 640), (700, 3, 9000), (390, 7, 4096)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_segments(dev, dtype, T, B, D):
    print(f"gated segments {T}x{B}x{D} {dtype}", flush=True)
    x, gate, h0, st, dh, dend = inputs(T, B, D, dtype, dev, "sigmoid", True, seed=2, shift=4.0)
    for s in (None, st):
        check(run(x, gate, h0, s, "sigmoid", True, dh, dend), reference(x, gate, h0, s, "sigmoid", True, dh, dend))


@pytest.mark.parametrize("which", ["h", "end", "no_h0"])
@pytest.mark.parametrize("T", [3, 700])
def test_parts_of_the_gradient(dev, which, T):
    x, gate, h0, st, dh, dend = inputs(T, 2, 70, torch.float32, dev, "log", True, seed=3)
    dh, dend = None if which == "end" else dh, None if which == "h" else dend
    h0 = None if which == "no_h0" else h0
    check(run(x, gate, h0, st, "log", True, dh, dend), reference(x, gate, h0, st, "log", True, dh, dend))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["projection", "batch_major", "odd_offset", "last_axis", "expanded", "one_row_in_odd_memory"])
def test_layouts(dev, dtype, layout):
    from lifscan import hip_gated as G
    T, B, D = (1 if layout == "one_row_in_odd_memory" else 150), 2, 64
    x, gate, h0, st, dh, dend = inputs(T, B, D, dtype, dev, seed=4)
    if layout == "projection":
        x, gate = torch.cat([x, gate], -1).split(D, -1)
    elif layout == "batch_major":
        x, gate, dh = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, gate, dh))
    elif layout == "odd_offset":
        x, gate = (torch.cat([t[..., :1], t], -1)[..., 1:] for t in (x, gate))
    elif layout == "last_axis":
        x, gate, dh = (t.transpose(0, 2).contiguous().transpose(0, 2) for t in (x, gate, dh))
    elif layout == "expanded":
        gate, dh = gate[:, :1].expand(T, B, D), dh[:1].expand(T, B, D)
    else:
        x, gate = (torch.cat([t, t, t], -1)[..., :D + 1].contiguous()[..., :D] for t in (x, gate))
    ins = [t.detach().requires_grad_(True) for t in (x, gate, h0)]
    h, end = G.gated_scan(*ins, starts=st)
    assert h.is_contiguous()
    grads = torch.autograd.grad((h, end), ins, (dh, dend))
    want = reference(x, gate, h0, st, "sigmoid", True, dh, dend)
    check({"h": h, "end": end, **dict(zip(("dx", "dgate", "dh0"), grads))}, want)


def test_training_copies_an_operand_once(dev):
    """Operands whose last axis is not contiguous, and strided starts, are laid out once a call, and their gradients
    reach the tensors that were given."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Copies(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.n += func.overloadpacket in (torch.ops.aten.clone, torch.ops.aten.copy_)
            return func(*args, **(kwargs or {}))

    from lifscan import hip_gated as G
    x, gate, h0, starts, dh, dend = inputs(40, 3, 32, torch.float32, dev, starts=True, seed=31)
    want = run(x, gate, h0, starts, "sigmoid", True, dh, dend)
    a, b = (t.transpose(0, 2).contiguous().transpose(0, 2).requires_grad_(True) for t in (x, gate))
    late = starts.t().contiguous().t()
    for train in (True, False):
        with torch.set_grad_enabled(train), Copies() as seen:
            h, end = G.gated_scan(a, b, h0, starts=late)
        assert seen.n == 3, (train, seen.n)
        assert torch.equal(h, want["h"]) and torch.equal(end, want["end"])
        if train:
            for got, name in zip(torch.autograd.grad((h, end), (a, b), (dh, dend)), ("dx", "dgate")):
                assert torch.equal(got, want[name])


def test_starts_of_either_type_and_any_stride(dev):
    from lifscan import hip_gated as G
    x, gate, h0, st, *_ = inputs(40, 3, 16, torch.float32, dev, starts=True, seed=5)
    h, end = G.gated_scan(x, gate, h0, starts=st)
    for other in (st.to(torch.uint8) * 5, st.t().contiguous().t(), torch.stack([st, ~st], -1)[..., 0]):
        again = G.gated_scan(x, gate, h0, starts=other)
        assert torch.equal(again[0], h) and torch.equal(again[1], end)


@pytest.mark.parametrize("T", [60, 900])
def test_starts_drop_what_was_before(dev, T):
    """Packed sequences are those sequences one by one, and nothing that one holds reaches the next or the one
    before: not an infinity, not a NaN."""
    from lifscan import hip_gated as G
    B, D, cut = 2, 64, T // 3
    x, gate, h0, _, dh, dend = inputs(T, B, D, torch.float32, dev, seed=6)
    st = torch.zeros(T, B, dtype=torch.bool, device=dev)
    st[cut] = True
    want = run(x, gate, h0, st, "sigmoid", True, dh, dend)
    tail = run(x[cut:], gate[cut:], None, None, "sigmoid", True, dh[cut:], dend)
    ref = reference(x[cut:], gate[cut:], None, None, "sigmoid", True, dh[cut:], dend)
    for k in ("h", "dx", "dgate"):
        close(want[k][cut:], ref[k], k)
        close(tail[k], ref[k], k)
    for bad in (float("inf"), float("nan")):
        for where in ("x", "gate", "h0", "dh"):
            xs, gs, hs, ds = x.clone(), gate.clone(), h0.clone(), dh.clone()
            {"x": xs, "gate": gs, "h0": hs, "dh": ds}[where].view(-1, D)[:, 5] = bad if where != "dh" else 0.0
            if where == "dh":
                ds[cut:, :, 5] = bad
            else:
                for t, o in ((xs, x), (gs, gate)):
                    t[cut:] = o[cut:]
            clean = want
            if where == "dh":  # rows before the start as here, those behind it without the bad values
                zeros = ds.clone()
                zeros[cut:, :, 5] = 0.0
                clean = run(x, gate, h0, st, "sigmoid", True, zeros, dend)
            got = run(xs, gs, hs, st, "sigmoid", True, ds, dend)
            keep = slice(0, cut) if where == "dh" else slice(cut, T)
            names = ("dx", "dgate") if where == "dh" else ("h", "dx", "dgate")
            for k in names:
                assert torch.equal(got[k][keep], clean[k][keep]), (where, bad, k)
            others = [d for d in range(D) if d != 5]
            assert torch.equal(got["h"][..., others], want["h"][..., others])
            if where != "dh":
                assert torch.equal(got["end"], want["end"])


def test_values_that_are_not_finite_reach_later_rows_of_their_channel(dev):
    from lifscan import hip_gated as G
    T, B, D = 400, 2, 66
    x, gate, h0, *_ = inputs(T, B, D, torch.float32, dev, seed=7)
    h, end = G.gated_scan(x, gate, h0)
    for bad in (float("inf"), float("-inf"), float("nan")):
        xs = x.clone()
        xs[150, 1, 7] = bad
        got, last = G.gated_scan(xs, gate, h0)
        assert not bool(got[150:, 1, 7].isfinite().any()) and not bool(last[1, 7].isfinite())
        mask = torch.ones_like(got, dtype=torch.bool)
        mask[150:, 1, 7] = False
        assert torch.equal(got[mask], h[mask])
    gs = gate.clone()
    gs[150, 1, 7] = float("nan")
    got, _ = G.gated_scan(x, gs, h0)
    assert bool(got[150:, 1, 7].isnan().all()) and torch.equal(got[:150], h[:150])


@pytest.mark.parametrize("decay", ["sigmoid", "log"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gates_at_the_ends(dev, decay, dtype):
    """Decays of exactly 0 and 1, close to either, and log decays above 0, which count as 0."""
    inf = float("inf")
    values = [-inf, -1000.0, -104.0, -89.0, -30.0, -1.0, -0.35, -0.34, -1e-3, -1e-7, 0.0, 1e-7, 0.5, 20.0, 30.0, 89.0, 104.0, 1000.0, inf]
    gate = torch.tensor(values, dtype=torch.float64).repeat(5)[:, None, None].expand(-1, 1, len(values)).clone()
    gate = torch.stack([gate[:, :, i].roll(i, 0) for i in range(len(values))], -1).to(dtype).to(dev)
    T, B, D = gate.shape
    x, _, h0, _, dh, dend = inputs(T, B, D, dtype, dev, seed=8)
    for mix in (True, False):
        got = run(x, gate, h0, None, decay, mix, dh, dend)
        # the smallest normal number stands for zero where the hardware's power of two gives it
        want = reference(x, gate, h0, None, decay, mix, dh, dend)
        check(got, {k: (v, b + 2.0 ** -120) for k, (v, b) in want.items()})


def test_gradients_against_differences(dev):
    """Central differences along random directions: the sum of the outputs in 64 bits is accurate to about
    T*F of its terms' sum, divided by the step 2^-7; the third derivative adds some 2^-14."""
    from lifscan import hip_gated as G
    T, B, D = 90, 2, 20
    for decay, mix in FORMS:
        x, gate, h0, st, dh, dend = inputs(T, B, D, torch.float32, dev, decay, True, seed=9, shift=1.0)
        got = run(x, gate, h0, st, decay, mix, dh, dend)
        value = lambda *a: float((G.gated_scan(*a, starts=st, decay=decay, mix=mix)[0].double() * dh.double()).sum()  # noqa: E731
                                 + (G.gated_scan(*a, starts=st, decay=decay, mix=mix)[1].double() * dend.double()).sum())
        for i, k in enumerate(("dx", "dgate", "dh0")):
            v = torch.randn_like((x, gate, h0)[i])
            if decay == "log" and i == 1:
                v = v * gate  # stays below 0
            step = 2.0 ** -7
            at = lambda s: [t + s * step * v if j == i else t for j, t in enumerate((x, gate, h0))]  # noqa: E731
            diff = (value(*at(1)) - value(*at(-1))) / (2 * step)
            want = float((got[k].double() * v.double()).sum())
            size = float((got[k].double() * v.double()).abs().sum()) + 1e-3 * float(dh.abs().sum())
            assert abs(diff - want) <= 2.0 ** -9 * size, (decay, mix, k, diff, want, size)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 7), (2, 64), (65, 130), (5, 4096)])
def test_single_tokens_follow_the_recurrence(dev, dtype, B, D):
    from lifscan import hip_gated as G
    for decay, mix in FORMS:
        x, gate, h0, *_ = inputs(6, B, D, dtype, dev, decay, seed=10)
        state = h0.clone()
        want = reference(x, gate, h0, None, decay, mix)
        for t in range(6):
            h = G.gated_scan_step(x[t], gate[t], state, decay=decay, mix=mix)
            assert h.dtype == dtype
            close(h, (want["h"][0][t], want["h"][1][t]))
        close(state, want["end"])


def test_steps_read_views_and_continue_a_prompt(dev):
    from lifscan import hip_gated as G
    T, B, D = 70, 3, 96
    x, gate, h0, *_ = inputs(T, B, D, torch.bfloat16, dev, seed=11)
    both = torch.cat([x, gate], -1)
    want = reference(x, gate, h0, None, "sigmoid", True)
    h, state = G.gated_scan(x[:50], gate[:50], h0)
    for t in range(50, T):
        xs, gs = both[t].split(D, -1)
        h = G.gated_scan_step(xs, gs, state)
        close(h, (want["h"][0][t], want["h"][1][t]))
    close(state, want["end"])
    odd = torch.cat([both[0, :, :1], both[0]], -1)[:, 1:]
    a, b = h0.clone(), h0.clone()
    assert torch.equal(G.gated_scan_step(*both[0].split(D, -1), a), G.gated_scan_step(*odd.split(D, -1), b))
    assert torch.equal(a, b)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("B,D", [(1, 1000), (64, 1000), (37, 61)])
def test_steps_whose_operands_share_memory_with_the_state(dev, B, D, graph):
    """Values and gates are those from before the call, whichever part of the state, or more, they are views of."""
    from lifscan import hip_gated as G
    g = torch.Generator().manual_seed(B)
    start = torch.randn(B * D + 2 * D + 5, generator=g).to(dev)
    other = torch.randn(B, D, generator=g).to(dev)
    forms = {
        "one row": lambda s: s[D:2 * D].view(1, D).expand(B, D), "itself": lambda s: s[D:D + B * D].view(B, D),
        "one value": lambda s: s[D + 3:D + 4].view(1, 1).expand(B, D), "a shift behind": lambda s: s[D + 5:D + 5 + B * D].view(B, D),
        "a row before": lambda s: s[:B * D].view(B, D), "halves": lambda s: s.view(torch.bfloat16)[2 * D:2 * D + B * D].view(B, D),
        "its end": lambda s: s[B * D + D - 1:B * D + 2 * D - 1].view(1, D).expand(B, D),
        "columns": lambda s: s[D:D + B * D].view(D, B).t(), "every other": lambda s: s[D:D + B].view(B, 1).expand(B, D),
    }
    for name, of in forms.items():
        for which in ("x", "gate", "both"):
            buf, want = start.clone(), start.clone()
            held = of(want).clone()
            rest = other.to(held.dtype)
            at = lambda b: b[D:D + B * D].view(B, D)  # noqa: E731
            views = lambda v: (v if which != "gate" else rest, v if which != "x" else rest)  # noqa: E731
            h_want = G.gated_scan_step(*views(held), at(want))
            if graph:
                captured, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
                torch.cuda.synchronize()
                with torch.cuda.graph(captured, stream=side):
                    h = G.gated_scan_step(*views(of(buf)), at(buf))
                for _ in range(2):
                    buf.copy_(start)
                    captured.replay()
                torch.cuda.synchronize()
            else:
                h = G.gated_scan_step(*views(of(buf)), at(buf))
            # as bits: halves of fp32 numbers may be NaN
            bits = torch.int16 if h.dtype == torch.bfloat16 else torch.int32
            assert torch.equal(h.view(bits), h_want.view(bits)) and torch.equal(buf.view(torch.int32), want.view(torch.int32)), \
                (name, which)


def test_steps_whose_operands_lie_beside_the_state_are_not_copied(dev):
    from lifscan import hip_gated as G
    B, D = 5, 64
    buf = torch.randn(3 * B * D, device=dev)
    x, state, gate = (t.view(B, D) for t in buf.split(B * D))
    G.gated_scan_step(x, gate, state)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    h = G.gated_scan_step(x, gate, state)
    assert torch.cuda.max_memory_allocated() - before <= max(512, -(-h.nbytes // 512) * 512)


def test_no_rows_no_batch(dev):
    from lifscan import hip_gated as G
    x = torch.zeros(0, 3, 8, device=dev, requires_grad=True)
    h0 = torch.randn(3, 8, device=dev, requires_grad=True)
    h, end = G.gated_scan(x, x, h0)
    assert h.shape == (0, 3, 8) and torch.equal(end, h0)
    d = torch.randn_like(h0)
    dx, dh0 = torch.autograd.grad(end, (x, h0), d)
    assert dx.shape == x.shape and torch.equal(dh0, d)
    h, end = G.gated_scan(x.detach(), x.detach())
    assert end.shape == (3, 8) and not bool(end.any())
    y = torch.zeros(4, 0, 8, device=dev, requires_grad=True)
    h, end = G.gated_scan(y, y)
    assert h.shape == (4, 0, 8) and end.shape == (0, 8)
    assert torch.autograd.grad(h.sum(), y)[0].shape == y.shape
    assert G.gated_scan_step(y[0].detach(), y[0].detach(), torch.zeros(0, 8, device=dev)).shape == (0, 8)


def test_offsets_beyond_32_bits(dev):
    """Rows that lie 2^31 elements apart."""
    from lifscan import hip_gated as G
    T, B, D = 3, 1, 64
    x, gate, h0, _, dh, dend = inputs(T, B, D, torch.bfloat16, dev, seed=12)
    far = torch.empty(2 ** 32 + 2 ** 20, dtype=torch.bfloat16, device=dev)
    views = far.as_strided((T, B, D), (2 ** 31, D, 1)), far.as_strided((T, B, D), (2 ** 31, D, 1), 4096)
    views[0].copy_(x), views[1].copy_(gate)
    got = run(*views, h0, None, "sigmoid", True, dh, dend)
    want = run(x, gate, h0, None, "sigmoid", True, dh, dend)
    for k in got:
        assert torch.equal(got[k], want[k])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_batches_beyond_32_bits(dev, dtype):
    """Batches of which a wave holds several, 2^32 bytes and more apart: no 32-bit offset reaches from one to
    the next."""
    T, B, D = 300, 2, 32
    x, gate, h0, st, dh, dend = inputs(T, B, D, dtype, dev, starts=True, seed=16)
    apart = 2 ** 32 // x.element_size() + 2 ** 20
    far = torch.empty(apart + 2 ** 20, dtype=dtype, device=dev)
    views = [far.as_strided((T, B, D), (D, apart, 1), i * T * D) for i in range(3)]
    for v, t in zip(views, (x, gate, dh)):
        v.copy_(t)
    got = run(views[0], views[1], h0, st, "sigmoid", True, views[2], dend)
    check(got, reference(x, gate, h0, st, "sigmoid", True, dh, dend))


def test_one_tensor_as_value_and_gate(dev):
    from lifscan import hip_gated as G
    x, _, h0, _, dh, _ = inputs(200, 2, 24, torch.float32, dev, seed=17)
    y = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(G.gated_scan(y, y, h0)[0], y, dh)
    want = reference(x, x, h0, None, "sigmoid", True, dh)
    close(got, (want["dx"][0] + want["dgate"][0], want["dx"][1] + want["dgate"][1] + F * (want["dx"][0].abs() + want["dgate"][0].abs())))
    # a gradient for one of them alone
    for i in range(3):
        ins = [x.clone(), x.clone(), h0.clone()]
        ins[i].requires_grad_(True)
        (got,) = torch.autograd.grad(G.gated_scan(*ins)[0], ins[i], dh)
        close(got, want[("dx", "dgate", "dh0")[i]])


def test_calls_at_once_on_two_streams(dev):
    from lifscan import hip_gated as G
    a, b = (inputs(3000, 2, 96, torch.bfloat16, dev, starts=True, seed=s) for s in (18, 19))
    want = [run(*t[:4], "sigmoid", True, *t[4:]) for t in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for n in range(3):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = run(*t[:4], "sigmoid", True, *t[4:])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for k in w:
            assert torch.equal(g[k], w[k])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_same_bits_on_every_run_and_stream(dev, dtype):
    args = inputs(1500, 2, 200, dtype, dev, starts=True, seed=13)
    x, gate, h0, st, dh, dend = args
    first = run(x, gate, h0, st, "sigmoid", True, dh, dend)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(x, gate, h0, st, "sigmoid", True, dh, dend)
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], second[k])


def test_graph_replays(dev):
    """Forward, gradients and a step captured into one graph, replayed on new values between eager work."""
    from lifscan import hip_gated as G
    T, B, D = 700, 2, 128
    x, gate, h0, st, dh, dend = inputs(T, B, D, torch.bfloat16, dev, starts=True, seed=14)
    ins = [t.clone().requires_grad_(True) for t in (x, gate, h0)]
    state = torch.zeros(B, D, device=dev)

    def work():
        h, end = G.gated_scan(*ins, starts=st)
        grads = torch.autograd.grad((h, end), ins, (dh, dend))
        with torch.no_grad():
            one = G.gated_scan_step(ins[0][0], ins[1][0], state)
        return [h.detach(), end.detach(), *grads, one]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for n in range(3):
        nx, ngate, nh0, *_ = inputs(T, B, D, torch.bfloat16, dev, seed=20 + n)
        with torch.no_grad():
            for t, v in zip(ins, (nx, ngate, nh0)):
                t.copy_(v)
            state.copy_(nh0)
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        with torch.no_grad():
            state.copy_(nh0)
        for a, b in zip(kept, work()):
            assert torch.equal(a, b)


def test_a_state_changed_in_place_is_noticed(dev):
    from lifscan import hip_gated as G
    x = torch.randn(2, 8, device=dev)
    state = torch.randn(2, 8, device=dev)
    w = torch.randn(2, 8, device=dev, requires_grad=True)
    y = (w * state).sum()
    G.gated_scan_step(x, x, state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():
        s = torch.zeros(2, 8, device=dev)
        G.gated_scan_step(x, x, s)
        assert bool(s.any())


def test_saved_tensors_that_come_back_changed(dev):
    from lifscan import hip_gated as G
    x, gate, h0, st, dh, dend = inputs(300, 2, 64, torch.float32, dev, starts=True, seed=15)
    want = run(x, gate, h0, st, "sigmoid", True, dh, dend)

    def back(t):  # not contiguous, elsewhere
        return torch.stack([t, t], -1)[..., 0] if t.dim() else t

    ins = [t.clone().requires_grad_(True) for t in (x, gate, h0)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        h, end = G.gated_scan(*ins, starts=st)
    for a, k in zip(torch.autograd.grad((h, end), ins, (dh, dend)), ("dx", "dgate", "dh0")):
        assert torch.equal(a, want[k])
    for change in (lambda t: t[:1], lambda t: t.half(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            h, end = G.gated_scan(*ins, starts=st)
        with pytest.raises((ValueError, RuntimeError)):
            torch.autograd.grad((h, end), ins, (dh, dend))


def test_refusals(dev):
    from lifscan import hip_gated as G
    x = torch.randn(4, 2, 8, device=dev)
    s = torch.zeros(2, 8, device=dev)
    st = torch.zeros(4, 2, dtype=torch.bool, device=dev)
    bad = [lambda: G.gated_scan(x[0], x[0]), lambda: G.gated_scan(x, x[:3]), lambda: G.gated_scan(x, x.half()),
           lambda: G.gated_scan(x.double(), x.double()), lambda: G.gated_scan(x.cpu(), x.cpu()),
           lambda: G.gated_scan(x, x, s[:1]), lambda: G.gated_scan(x, x, s.half()), lambda: G.gated_scan(x, x, s.cpu()),
           lambda: G.gated_scan(x, x, s, starts=st[:3]), lambda: G.gated_scan(x, x, s, starts=st.float()),
           lambda: G.gated_scan(x, x, s, starts=st.cpu()), lambda: G.gated_scan(x, x, decay="tanh"),
           lambda: G.gated_scan(x[..., :0], x[..., :0]), lambda: G.gated_scan(torch._neg_view(x), x),
           lambda: G.gated_scan_step(x, x, s), lambda: G.gated_scan_step(x[0], x[0], s.t().contiguous().t()),
           lambda: G.gated_scan_step(x[0], x[0], s.half()), lambda: G.gated_scan_step(x[0], x[0], s[:1]),
           lambda: G.gated_scan_step(x[0].clone().requires_grad_(True), x[0], s),
           lambda: G.gated_scan_step(x[0], x[0], s, decay=0)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    assert not bool(s.any())
    y = x.clone().requires_grad_(True)
    h, _ = G.gated_scan(y, x)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(h.sum(), y, create_graph=True)


def test_forward_mode_and_traces_are_refused(dev):
    import torch.autograd.forward_ad as fw
    from lifscan import hip_gated as G
    x, s = torch.randn(4, 2, 8, device=dev), torch.zeros(2, 8, device=dev)
    for f, args in ((lambda *a: G.gated_scan(*a)[0], (x, x, s)), (lambda *a: G.gated_scan_step(*a), (x[0], x[0], s))):
        for i in range(len(args)):
            with fw.dual_level():
                duals = [fw.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*duals)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, args, check_trace=False)
    y = x.clone().requires_grad_(True)
    h, _ = G.gated_scan(y, x)
    g = torch.randn_like(h)
    (want,) = torch.autograd.grad(h, y, -g, retain_graph=True)
    (got,) = torch.autograd.grad(h, y, torch._neg_view(g))
    assert torch.equal(got, want)
