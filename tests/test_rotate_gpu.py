"""GPU: norms of queries and keys for each head and their rotation by position (lifscan.hip_linattn.norm_rotate)
against the definition in 64 bits, the gradients against the written-out formulas in 64 bits and against
differences.

Tolerances.  Results are rounded once to their type (u = 2^-24, 2^-8, 2^-11) after fp32 arithmetic: sums of up
to 256 terms in a tree of 8 values a lane and at most 5 steps, a root of 1 ulp, and a cosine and a sine that
are off by 3 * 2^-24 at most (the angle's rounding, half a turn's eighth at most 2^-25; the sums' four steps).
So an element is off by u of itself and 64 * 2^-24 of the magnitude that the same formula gives with every
part's absolute value; sums over n rows add n * 2^-24 of theirs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def freqs(rot, dev, base=10000.0):
    return (base ** -(torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))).to(dev)


def reference(x, w, positions, inv_freq, eps, pairs, g=None):
    """(y, its magnitude), and with g (dx, magnitude), (dw, magnitude): 64 bits on the CPU."""
    x = x.detach().double().cpu()
    D = x.shape[-1]
    half = 0 if inv_freq is None else inv_freq.numel()
    i = torch.arange(half)
    first, second = (i, i + half) if pairs == "halves" else (2 * i, 2 * i + 1)
    if half:
        p = positions.cpu().double()
        p = p if p.dim() == x.dim() - 2 else p[:, None].expand(x.shape[:2])
        angle = p[..., None, None] * inv_freq.cpu().double()
        c, s = angle.cos(), angle.sin()

    def turn(y, sign, size=False):
        z = y.clone()
        if half:
            u, v = y[..., first], y[..., second]
            if size:
                z[..., first], z[..., second] = u * c.abs() + v * s.abs() + 0.1 * (u + v), v * c.abs() + u * s.abs() + 0.1 * (u + v)
            else:
                z[..., first], z[..., second] = u * c - sign * v * s, v * c + sign * u * s
        return z

    mean = lambda t: t.sum(-1, keepdim=True) / D  # noqa: E731
    if w is None:
        r, w = torch.ones_like(x[..., :1]), torch.ones(D, dtype=torch.float64)
        norm = False
    else:
        r, w, norm = (mean(x * x) + eps).pow(-0.5), w.detach().double().cpu(), True
    y = x * r * w
    out = {"y": (turn(y, 1), turn(y.abs(), 1, True))}
    if g is not None:
        u, ua = turn(g.double().cpu(), -1), turn(g.double().cpu().abs(), -1, True)
        if norm:
            m, ma = u * w, ua * w.abs()
            out["dx"] = r * (m - x * r * r * mean(m * x)), r * (ma + x.abs() * r * r * mean(ma * x.abs()))
            dims = tuple(range(x.dim() - 1))
            out["dw"] = (u * x * r).sum(dims), (ua * x.abs() * r).sum(dims)
        else:
            out["dx"] = u, ua
    return out


def close(got, want, n=64):
    value, size = want
    assert tuple(got.shape) == tuple(value.shape)
    err = (got.detach().double().cpu() - value).abs()
    bound = U[got.dtype] * value.abs() + n * F * size + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126)
    assert bool((err <= bound).all()), float((err / bound).max())


def inputs(lead, H, HK, D, dtype, dev, norm=True, far=0, seed=0):
    g = torch.Generator().manual_seed(seed + D + 100 * H)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, gq, gk = mk(*lead, H, D), mk(*lead, HK, D), mk(*lead, H, D), mk(*lead, HK, D)
    wq, wk = (1 + 0.2 * mk(D), 1 + 0.2 * mk(D)) if norm else (None, None)
    pos = torch.randint(0, 50 + far, tuple(lead), generator=g) if lead else None
    return [t.to(dtype).to(dev) for t in (q, k, gq, gk)] + [t.to(dev) if t is not None else None for t in (wq, wk, pos)]


def run(q, k, wq, wk, pos, f, pairs, gq=None, gk=None, eps=1e-6):
    from lifscan import hip_linattn as LA
    ins = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, wq, wk)]
    yq, yk = LA.norm_rotate(ins[0], ins[1], pos, f, ins[2], ins[3], eps=eps, pairs=pairs)
    got = {"q": yq, "k": yk}
    outs = [(o, g) for o, g in ((yq, gq), (yk, gk)) if g is not None]
    have = [t for t in ins if t is not None]
    if outs:
        grads = iter(torch.autograd.grad([o for o, _ in outs], have, [g for _, g in outs], allow_unused=True))
        got.update((n, next(grads)) for n, t in zip(("dq", "dk", "dwq", "dwk"), ins) if t is not None)
    return got


def check(got, q, k, wq, wk, pos, f, pairs, gq, gk, eps=1e-6):
    for name, x, w, g in (("q", q, wq, gq), ("k", k, wk, gk)):
        want = reference(x, w, pos, f, eps, pairs, g)
        close(got[name], want["y"])
        if g is not None:
            close(got["d" + name], want["dx"])
            if w is not None:
                close(got["dw" + name], want["dw"], 64 + x.numel() // x.shape[-1])


CASES = [((1, 1), 1, 1, 2, 2), ((3, 2), 2, 1, 8, 8), ((5, 1), 3, 3, 16, 4), ((7, 3), 4, 2, 32, 32), ((2, 5), 6, 2, 64, 64),
         ((9, 2), 5, 1, 64, 24), ((4, 4), 7, 7, 80, 36), ((3, 3), 16, 4, 128, 128), ((5, 2), 3, 1, 128, 64),
         ((2, 3), 9, 3, 256, 256), ((3, 1), 5, 2, 250, 122), ((2, 2), 3, 1, 254, 254), ((6, 1), 2, 2, 66, 66), ((4, 2), 2, 1, 96, 0),
         ((11,), 8, 8, 64, 64), ((5,), 5, 1, 74, 10)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lead,H,HK,D,rot", CASES)
def test_forward_and_gradients(dev, dtype, lead, H, HK, D, rot):
    print(f"rotate {lead} {H}/{HK} heads of {D}, {rot} rotated, {dtype}", flush=True)
    for pairs in ("halves", "neighbours"):
        for norm in (True, False):
            q, k, gq, gk, wq, wk, pos = inputs(lead, H, HK, D, dtype, dev, norm)
            f = freqs(rot, dev) if rot else None
            got = run(q, k, wq, wk, pos if rot else None, f, pairs, gq, gk)
            assert got["q"].dtype == got["dq"].dtype == dtype
            check(got, q, k, wq, wk, pos, f, pairs, gq, gk)


@pytest.mark.parametrize("D,rot,dtype", [(64, 64, torch.bfloat16), (128, 96, torch.float32), (80, 36, torch.float16),
                                         (256, 256, torch.bfloat16)])
def test_many_tokens(dev, D, rot, dtype):
    """More items than workgroups of the gradients: sums are carried over; heads split over several waves."""
    T, B, H, HK = 1700, 3, 6, 3
    q, k, gq, gk, wq, wk, _ = inputs((T, B), H, HK, D, dtype, dev)
    pos, f = torch.arange(T, device=dev), freqs(rot, dev)
    check(run(q, k, wq, wk, pos, f, "halves", gq, gk), q, k, wq, wk, pos, f, "halves", gq, gk)


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 31, 2 ** 40])
def test_far_and_negative_positions(dev, far):
    """fp32 would keep 2^-4 of a radian at 2^20.  Beyond that the frequency's own last place in 64 bits counts:
    position * 2^-52 radians more."""
    q, k, *_ , wq, wk, pos = inputs((40, 2), 2, 2, 64, torch.float32, dev, far=0)
    f = freqs(64, dev)
    for p in (pos + far, -(pos + far)):
        for t, w in ((q, wq), (k, wk)):
            y, size = reference(t, w, p, f, 1e-6, "halves")["y"]
            got = run(q, k, wq, wk, p, f, "halves")["q" if t is q else "k"]
            err = (got.detach().double().cpu() - y).abs()
            assert bool((err <= F * y.abs() + (64 * F + 4 * far * 2.0 ** -52) * size).all())


def test_positions_of_any_form(dev):
    from lifscan import hip_linattn as LA
    T, B = 9, 4
    q, k, *_, wq, wk, pos = inputs((T, B), 2, 1, 32, torch.float32, dev)
    f = freqs(32, dev)
    want = LA.norm_rotate(q, k, pos, f, wq, wk)
    for p in (pos.int(), pos.t().contiguous().t(), torch.stack([pos, pos + 1], -1)[..., 0]):
        for a, b in zip(LA.norm_rotate(q, k, p, f, wq, wk), want):
            assert torch.equal(a, b)
    row = pos[:, 0].contiguous()
    want = LA.norm_rotate(q, k, row[:, None].expand(T, B), f, wq, wk)
    for a, b in zip(LA.norm_rotate(q, k, row, f, wq, wk), want):
        assert torch.equal(a, b)
    # one token each: as a row of a sequence
    for a, b in zip(LA.norm_rotate(q[3], k[3], pos[3], f, wq, wk), LA.norm_rotate(q, k, pos, f, wq, wk)):
        assert torch.equal(a, b[3])
    # frequencies and weights of other types
    f32 = f.float()
    for a, b in zip(LA.norm_rotate(q, k, pos, f32, wq, wk), LA.norm_rotate(q, k, pos, f32.double(), wq, wk)):
        assert torch.equal(a, b)
    w = wq.bfloat16()
    for a, b in zip(LA.norm_rotate(q, k, pos, f, w, wk), LA.norm_rotate(q, k, pos, f, w.float(), wk)):
        assert torch.equal(a, b)


def test_positions_are_relative(dev):
    """What the rotation is for: products of a query and a key depend on their distance alone."""
    from lifscan import hip_linattn as LA
    q = torch.randn(1, 1, 1, 64, device=dev).expand(20, 1, 1, 64)
    f = freqs(64, dev)
    at = torch.arange(20, device=dev)
    for pairs in ("halves", "neighbours"):
        y, z = LA.norm_rotate(q, q, at + 1000003, f, pairs=pairs)
        dots = (y[5:, 0, 0].double() * z[:15, 0, 0].double()).sum(-1)
        assert float((dots - dots[0]).abs().max()) <= 64 * 64 * F * float((q[0] ** 2).sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["projection", "batch_major", "odd_offset", "last_axis", "expanded"])
def test_layouts(dev, dtype, layout):
    T, B, H, HK, D = 21, 3, 4, 2, 64
    q, k, gq, gk, wq, wk, pos = inputs((T, B), H, HK, D, dtype, dev)
    f = freqs(48, dev)
    if layout == "projection":
        both = torch.cat([q.flatten(-2), k.flatten(-2)], -1).split([H * D, HK * D], -1)
        q, k = both[0].unflatten(-1, (H, D)), both[1].unflatten(-1, (HK, D))
    elif layout == "batch_major":
        q, k, gq, gk = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, gq, gk))
    elif layout == "odd_offset":
        q, k, gq = (torch.cat([t[..., :1], t], -1)[..., 1:] for t in (q, k, gq))
    elif layout == "last_axis":
        q, k, gk = (t.transpose(0, 3).contiguous().transpose(0, 3) for t in (q, k, gk))
    else:
        k, gq, gk = k[:, :1].expand(T, B, HK, D), gq[..., :1].expand(T, B, H, D), gk[:1, :, :1].expand(T, B, HK, D)
    got = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    assert got["q"].is_contiguous() and got["k"].is_contiguous()
    check(got, q, k, wq, wk, pos, f, "halves", gq, gk)


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("norm", [True, False])
def test_one_output_alone(dev, which, norm):
    q, k, gq, gk, wq, wk, pos = inputs((30, 2), 4, 2, 64, torch.float32, dev, norm)
    f = freqs(64, dev)
    gq, gk = (gq, None) if which == "q" else (None, gk)
    got = run(q, k, wq, wk, pos, f, "neighbours", gq, gk)
    check(got, q, k, wq, wk, pos, f, "neighbours", gq, gk)
    other = "k" if which == "q" else "q"
    assert got["d" + other] is None or not bool(got["d" + other].any())
    if norm:
        assert got["dw" + other] is None or not bool(got["dw" + other].any())


def test_weights_that_ask_for_no_gradient(dev):
    from lifscan import hip_linattn as LA
    q, k, gq, gk, wq, wk, pos = inputs((30, 2), 4, 2, 64, torch.float32, dev)
    f = freqs(64, dev)
    want = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    for which in ("", "q", "k"):
        a, b, u, v = (t.clone() for t in (q, k, wq, wk))
        a.requires_grad_(True), b.requires_grad_(True)
        ins, names = [a, b], ["dq", "dk"]
        if which:
            ins.append((u if which == "q" else v).requires_grad_(True))
            names.append("dw" + which)
        y, z = LA.norm_rotate(a, b, pos, f, u, v)
        for got, n in zip(torch.autograd.grad((y, z), ins, (gq, gk)), names):
            assert torch.equal(got, want[n])
        if not which:  # the weights' alone
            u.requires_grad_(True), v.requires_grad_(True)
            y, z = LA.norm_rotate(q, k, pos, f, u, v)
            for got, n in zip(torch.autograd.grad((y, z), (u, v), (gq, gk)), ("dwq", "dwk")):
                assert torch.equal(got, want[n])


def test_heads_of_zeros_and_large_eps(dev):
    q, k, gq, gk, wq, wk, pos = inputs((6, 2), 3, 1, 64, torch.float32, dev)
    q[2, 1] = 0.0
    f = freqs(64, dev)
    for eps in (1e-6, 0.5):
        got = run(q, k, wq, wk, pos, f, "halves", gq, gk, eps=eps)
        check(got, q, k, wq, wk, pos, f, "halves", gq, gk, eps=eps)
        assert not bool(got["q"][2, 1].any()) and bool(got["dq"].isfinite().all())


def test_values_that_are_not_finite_stay_in_their_head(dev):
    q, k, gq, gk, wq, wk, pos = inputs((6, 2), 3, 2, 64, torch.float32, dev)
    f = freqs(64, dev)
    want = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    q[4, 1, 2, 9] = float("nan")
    got = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    assert bool(got["q"][4, 1, 2].isnan().all()) and bool(got["dq"][4, 1, 2].isnan().all())
    mask = torch.ones(q.shape, dtype=torch.bool, device=dev)
    mask[4, 1, 2] = False
    for n in ("q", "dq"):
        assert torch.equal(got[n][mask], want[n][mask])
    assert torch.equal(got["k"], want["k"]) and torch.equal(got["dwk"], want["dwk"])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("D,rot", [(64, 0), (64, 24), (66, 2), (80, 36), (128, 64), (250, 122), (256, 8)])
def test_columns_that_pass_are_left_alone(dev, dtype, pairs, D, rot):
    """Whatever the columns behind the rotated ones hold: without a norm they come out as they went in, in both
    directions, and nothing of them reaches another column; with one, no other column's weight gets a gradient of it."""
    q, k, gq, gk, wq, wk, pos = inputs((7, 2), 3, 2, D, dtype, dev)
    f = freqs(rot, dev)
    odd = torch.tensor([float("inf"), float("nan"), -0.0, float("-inf")], device=dev).to(dtype)
    x, y = k.clone(), gk.clone()
    for t in (x, y):
        t[..., rot::3] = odd[torch.arange(t[..., rot::3].numel(), device=dev) % 4].view_as(t[..., rot::3])

    def same(a, b):
        assert bool(((a == b) & (torch.signbit(a) == torch.signbit(b)) | a.isnan() & b.isnan()).all())

    got = run(q, x, None, None, pos, f, pairs, gq, y)
    want = run(q, k, None, None, pos, f, pairs, gq, gk)
    for name, t in (("k", x), ("dk", y)):
        same(got[name][..., rot:], t[..., rot:])
        assert torch.equal(got[name][..., :rot], want[name][..., :rot])
    got = run(q, k, wq, wk, pos, f, pairs, gq, y)
    want = run(q, k, wq, wk, pos, f, pairs, gq, gk)
    others = torch.ones(D, dtype=torch.bool, device=dev)
    others[rot::3] = False
    assert torch.equal(got["dwk"][others], want["dwk"][others]) and torch.equal(got["dwq"], want["dwq"])
    assert not bool(got["dwk"][~y.isfinite().flatten(0, 2).all(0)].isfinite().any())



def test_the_weights_sums_do_not_drift(dev):
    """1280 workgroups' equal sums of 4 equal terms.  Doubled they stay exact, so what rounds is 2 of the 3 additions in a
    workgroup and as many as are made one after the other behind it: with 5 in a row and pairs from there on, 3.  Each is
    off by F of what it has summed, and each term by 2 F (a root of 1 ulp, a product): 7 F in all; 40 in a row and 32 in
    a row are off by up to 14 F."""
    T, D = 5120, 256
    g = torch.Generator().manual_seed(5)
    grads = [(1 + torch.rand(D, generator=g)).to(dev).expand(T, 1, 1, D) for _ in range(2)]
    x, w = torch.ones(T, 1, 1, D, device=dev), torch.ones(D, device=dev)
    got = run(x, x, w, w, None, None, "halves", *grads, eps=0.0)
    for name, t in zip(("dwq", "dwk"), grads):
        want = T * t[0, 0, 0].double()
        assert float(((got[name].double() - want).abs() / want).max()) <= 7 * F



def test_gradients_against_differences(dev):
    """Central differences of the 64-bit sum of fp32 outputs: with steps of 2^-6 the third derivative leaves
    some 2^-12 of the terms' sum, and the outputs' roundings 2^-24 of it over the step."""
    from lifscan import hip_linattn as LA
    q, k, gq, gk, wq, wk, pos = inputs((12, 2), 3, 1, 40, torch.float32, dev)
    f = freqs(28, dev)
    got = run(q, k, wq, wk, pos, f, "halves", gq, gk)

    def value(q, k, wq, wk):
        a, b = LA.norm_rotate(q, k, pos, f, wq, wk)
        return float((a.double() * gq.double()).sum() + (b.double() * gk.double()).sum())

    ins, step = [q, k, wq, wk], 2.0 ** -6
    for i, name in enumerate(("dq", "dk", "dwq", "dwk")):
        v = torch.randn_like(ins[i])
        at = lambda s: [t + s * step * v if j == i else t for j, t in enumerate(ins)]  # noqa: E731
        diff = (value(*at(1)) - value(*at(-1))) / (2 * step)
        want = float((got[name].double() * v.double()).sum())
        size = float((got[name].double() * v.double()).abs().sum())
        assert abs(diff - want) <= 2.0 ** -9 * size, (name, diff, want)


def test_empty(dev):
    from lifscan import hip_linattn as LA
    f = freqs(8, dev)
    w = torch.ones(8, device=dev, requires_grad=True)
    for lead in ((0, 3), (3, 0), (0,)):
        q = torch.zeros(*lead, 2, 8, device=dev, requires_grad=True)
        pos = torch.zeros(lead, dtype=torch.int64, device=dev)
        a, b = LA.norm_rotate(q, q, pos, f, w, w)
        assert a.shape == q.shape
        dq, dw = torch.autograd.grad(a.sum() + b.sum(), (q, w))
        assert dq.shape == q.shape and not bool(dw.any())
    q, k = torch.randn(3, 2, 0, 8, device=dev), torch.randn(3, 2, 1, 8, device=dev)
    pos = torch.zeros(3, dtype=torch.int64, device=dev)
    a, b = LA.norm_rotate(q, k, pos, f)
    assert a.shape == q.shape and torch.equal(b, k)
    # no queries, or neither: the others' gradients, and zeros for the weights
    q.requires_grad_(True), k.requires_grad_(True)
    g = torch.randn_like(k)
    v = torch.ones(8, device=dev, requires_grad=True)
    a, b = LA.norm_rotate(q, k, pos, f, v, w)
    dq, dk, dv, dw = torch.autograd.grad((a, b), (q, k, v, w), (torch.zeros_like(a), g))
    assert dq.shape == q.shape and not bool(dv.any())
    want = reference(k, w, pos, f, 1e-6, "halves", g)
    close(dk, want["dx"]), close(dw, want["dw"], 64 + 6)
    a, b = LA.norm_rotate(q, q, pos, f, v, w)
    dv, dw = torch.autograd.grad(a.sum() + b.sum(), (v, w))
    assert not bool(dv.any()) and not bool(dw.any())
    # frequencies of none are no rotation
    a, b = LA.norm_rotate(k, k, pos, f[:0])
    assert torch.equal(a, k) and torch.equal(b, k)


def test_offsets_beyond_32_bits(dev):
    from lifscan import hip_linattn as LA
    q, k, _, _, wq, wk, _ = inputs((3, 1), 2, 1, 64, torch.bfloat16, dev)
    f, pos = freqs(64, dev), torch.arange(3, device=dev)
    far = torch.empty(2 ** 32 + 2 ** 20, dtype=torch.bfloat16, device=dev)
    view = far.as_strided((3, 1, 2, 64), (2 ** 31, 128, 64, 1))
    view.copy_(q)
    for a, b in zip(LA.norm_rotate(view, k, pos, f, wq, wk), LA.norm_rotate(q, k, pos, f, wq, wk)):
        assert torch.equal(a, b)


def test_same_bits_on_every_run_stream_and_split(dev):
    q, k, gq, gk, wq, wk, pos = inputs((500, 2), 8, 2, 64, torch.bfloat16, dev)
    f = freqs(64, dev)
    first = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    torch.cuda.current_stream().wait_stream(side)
    for n in first:
        assert torch.equal(first[n], second[n])
    # a token's heads do not depend on how many tokens there are
    few = run(q[:2], k[:2], wq, wk, pos[:2], f, "halves", gq[:2], gk[:2])
    for n in ("q", "k", "dq", "dk"):
        assert torch.equal(few[n], first[n][:2])


def test_graph_replays(dev):
    from lifscan import hip_linattn as LA
    q, k, gq, gk, wq, wk, pos = inputs((64, 2), 4, 2, 64, torch.bfloat16, dev)
    f = freqs(64, dev)
    ins = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]

    def work():
        a, b = LA.norm_rotate(ins[0], ins[1], pos, f, ins[2], ins[3])
        return [a.detach(), b.detach(), *torch.autograd.grad((a, b), ins, (gq, gk))]

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
        with torch.no_grad():
            ins[0].normal_(), ins[1].normal_(), pos.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        for a, b in zip(kept, work()):
            assert torch.equal(a, b)


def test_saved_tensors_that_come_back_changed(dev):
    from lifscan import hip_linattn as LA
    q, k, gq, gk, wq, wk, pos = inputs((20, 2), 4, 2, 64, torch.float32, dev)
    f = freqs(64, dev)
    want = run(q, k, wq, wk, pos, f, "halves", gq, gk)
    ins = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0]):
        a, b = LA.norm_rotate(ins[0], ins[1], pos, f, ins[2], ins[3])
    for x, n in zip(torch.autograd.grad((a, b), ins, (gq, gk)), ("dq", "dk", "dwq", "dwk")):
        assert torch.equal(x, want[n])
    for change in (lambda t: t[:1], lambda t: t.half(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            a, b = LA.norm_rotate(ins[0], ins[1], pos, f, ins[2], ins[3])
        with pytest.raises((ValueError, RuntimeError)):
            torch.autograd.grad((a, b), ins, (gq, gk))


def test_refusals(dev):
    from lifscan import hip_linattn as LA
    q, k, _, _, wq, wk, pos = inputs((4, 2), 2, 1, 16, torch.float32, dev)
    f = freqs(16, dev)
    bad = [lambda: LA.norm_rotate(q.flatten(0, 2), k.flatten(0, 2), pos, f), lambda: LA.norm_rotate(q, k[:3], pos, f),
           lambda: LA.norm_rotate(q, k.half(), pos, f), lambda: LA.norm_rotate(q, k.cpu(), pos, f),
           lambda: LA.norm_rotate(q.double(), k.double(), pos, f), lambda: LA.norm_rotate(q[..., :15], k[..., :15], pos, f[:4]),
           lambda: LA.norm_rotate(q, k[..., :8], pos, f[:4]), lambda: LA.norm_rotate(q, k, None, f),
           lambda: LA.norm_rotate(q, k, pos, freqs(18, dev)), lambda: LA.norm_rotate(q, k, pos.float(), f),
           lambda: LA.norm_rotate(q, k, pos[:3], f), lambda: LA.norm_rotate(q, k, pos[0], f), lambda: LA.norm_rotate(q, k, pos.cpu(), f),
           lambda: LA.norm_rotate(q, k, pos, f.long()), lambda: LA.norm_rotate(q, k, pos, f.cpu()),
           lambda: LA.norm_rotate(q, k, pos, f, wq), lambda: LA.norm_rotate(q, k, pos, f, wq, wk[:8]),
           lambda: LA.norm_rotate(q, k, pos, f, wq, wk, eps=-1.0), lambda: LA.norm_rotate(q, k, pos, f, pairs="thirds"),
           lambda: LA.norm_rotate(q, k, pos, f.clone().requires_grad_(True)), lambda: LA.norm_rotate(torch._neg_view(q), k, pos, f),
           lambda: LA.norm_rotate(q[0], k[0], pos, f), lambda: LA.norm_rotate(q[0], k, pos, f)]
    wide = torch.zeros(2, 1, 1, 258, device=dev)
    bad.append(lambda: LA.norm_rotate(wide, wide))
    for fn in bad:
        with pytest.raises(ValueError):
            fn()
    y = q.clone().requires_grad_(True)
    a, _ = LA.norm_rotate(y, k, pos, f, wq, wk)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(a.sum(), y, create_graph=True)


def test_positions_and_frequencies_come_together(dev):
    from lifscan import hip_linattn as LA
    q, k, _, _, wq, wk, pos = inputs((4, 2), 2, 1, 16, torch.float32, dev)
    f = freqs(16, dev)
    for args in ((pos, None), (None, f), (pos, None, wq, wk), (pos.int(), None)):
        with pytest.raises(ValueError, match="inv_freq|positions"):
            LA.norm_rotate(q, k, *args)
    for a, b in zip(LA.norm_rotate(q, k), (q, k)):
        assert torch.equal(a, b)



def test_forward_mode_and_traces_are_refused(dev):
    import torch.autograd.forward_ad as fw
    from lifscan import hip_linattn as LA
    q, k, _, _, wq, wk, pos = inputs((4, 2), 2, 1, 16, torch.float32, dev)
    f = freqs(16, dev)
    call = lambda *a: LA.norm_rotate(a[0], a[1], pos, f, a[2], a[3])[0]  # noqa: E731
    args = (q, k, wq, wk)
    for i in range(4):
        with fw.dual_level():
            duals = [fw.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(call, args, check_trace=False)
    y = q.clone().requires_grad_(True)
    out = call(y, k, wq, wk)
    g = torch.randn_like(out)
    (want,) = torch.autograd.grad(out, y, -g, retain_graph=True)
    (got,) = torch.autograd.grad(out, y, torch._neg_view(g))
    assert torch.equal(got, want)
