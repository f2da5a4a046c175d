"""GPU: the row operators of a spiking language model (lifscan.hip_lm) against their definitions in 64
bits, their gradients against the written-out formulas in 64 bits and against differences.

Tolerances.  Results are rounded once to their type (u = 2^-24, 2^-8, 2^-11) after fp32 arithmetic, so an
element is off by at most u*|result| and a few dozen 2^-24 of the largest intermediate that enters it:
64 * 2^-24 times a magnitude that each test names.  Sums over n rows or terms add n * 2^-24 times the
sum of the terms' absolute values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F = 2.0 ** -24
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.float32, torch.bfloat16), (torch.float32, torch.float16)]
IDS = ["f32", "bf16", "f16", "f32+bf16", "f32+f16"]


def close(got, want, magnitude, n=64):
    assert tuple(got.shape) == tuple(want.shape)
    err = (got.detach().double().cpu() - want).abs()
    bound = U[got.dtype] * want.abs() + n * F * magnitude
    # the smallest steps of fp16 below its normal range
    bound = bound + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())


# ----------------------------------------------------------------------------- block_norm
def _bn_inputs(rows, D, tx, ty, dev, seed=0):
    g = torch.Generator().manual_seed(seed + D)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, y, gate = 2 * mk(rows, D), 0.5 * mk(rows, D), mk(rows, D)
    gx, gz = mk(rows, D), mk(rows, D)
    w_post, w_pre, a = 1 + 0.2 * mk(D), 1 + 0.2 * mk(D), 0.4 + 0.1 * mk(D)
    out = [x.to(tx), y.to(ty), gate.to(ty), w_post, w_pre, a, gx.to(tx), gz.to(ty)]
    return [t.to(dev) for t in out]


def bn_reference(x, y, gate, w_post, w_pre, a, eps, act, gx=None, gz=None):
    x, y, w_post, w_pre = (t.detach().double().cpu() for t in (x, y, w_post, w_pre))
    a = a.detach().double().cpu() if torch.is_tensor(a) else a
    D = x.shape[-1]
    if gate is None:
        f, df, sdf = torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x)
    else:
        gate = gate.detach().double().cpu()
        sg = 1 / (1 + torch.exp(-gate))
        f, df = (gate * sg, sg + gate * sg * (1 - sg)) if act == "silu" else (sg, sg * (1 - sg))
        sdf = sg + gate.abs() * sg * (1 - sg) if act == "silu" else df
    ry = (y.pow(2).sum(-1, keepdim=True) / D + eps).pow(-0.5)
    n = y * ry * w_post
    xn = x + a * f * n
    rx = (xn.pow(2).sum(-1, keepdim=True) / D + eps).pow(-0.5)
    out = {"x_new": xn, "z": xn * rx * w_pre}
    if gx is None and gz is None:
        return out
    gx = torch.zeros_like(x) if gx is None else gx.double().cpu()
    gz = torch.zeros_like(x) if gz is None else gz.double().cpu()
    mean = lambda t: t.sum(-1, keepdim=True) / D  # noqa: E731
    u = gz * w_pre
    dx = gx + rx * (u - xn * rx * rx * mean(u * xn))
    dh = a * dx
    m = dh * f * w_post
    out |= {"dx": dx, "dy": ry * (m - y * ry * ry * mean(m * y)), "dgate": dh * n * df}
    out |= {"dw_post": (dh * f * y * ry).sum(0), "dw_pre": (gz * xn * rx).sum(0), "da": (dx * f * n).sum(0)}
    # the same with every part's absolute value: what a rounding on the way is a share of
    a = abs(a) if not torch.is_tensor(a) else a.abs()
    u, f, n, xa, ya, w = (t.abs() for t in (u, f, n, x.abs() + (a * f * n).abs(), y, w_post))
    bx = gx.abs() + rx * (u + xa * rx * rx * mean(u * xa))
    bm = a * bx * f * w
    out["size"] = {"dx": bx, "dy": ry * (bm + ya * ry * ry * mean(bm * ya)), "dgate": a * bx * n * sdf,
                   "dw_post": (a * bx * f * ya * ry).sum(0), "dw_pre": (gz.abs() * xa * rx).sum(0),
                   "da": (bx * f * n).sum(0)}
    return out


def bn_run(x, y, gate, w_post, w_pre, a, eps, act, gx, gz):
    from lifscan import hip_lm as LM
    ins = [t.detach().requires_grad_(True) if torch.is_tensor(t) else None for t in (x, y, gate, w_post, w_pre, a)]
    scale = ins[5] if torch.is_tensor(a) else a
    x_new, z = LM.block_norm(ins[0], ins[1], ins[3], ins[4], gate=ins[2], res_scale=scale, eps=eps, act=act)
    outs = [(o, g) for o, g in ((x_new, gx), (z, gz)) if g is not None]
    have = [t for t in ins if t is not None]
    grads = iter(torch.autograd.grad([o for o, _ in outs], have, [g for _, g in outs], allow_unused=True))
    return {"x_new": x_new, "z": z, **{k: next(grads) if t is not None else None for k, t in
                                       zip(("dx", "dy", "dgate", "dw_post", "dw_pre", "da"), ins)}}


def bn_check(got, want, rows):
    for k in ("x_new", "z"):
        close(got[k], want[k], float(want[k].abs().max()) if want[k].numel() else 0.0)
    for k in ("dx", "dy", "dgate"):
        if got[k] is not None:
            close(got[k], want[k], want["size"][k])
    for k in ("dw_post", "dw_pre", "da"):
        if got[k] is not None:
            close(got[k], want[k], want["size"][k], n=64 + rows)


BN_SHAPES = [(1, 1), (3, 7), (5, 64), (2, 100), (33, 257), (700, 128), (4, 2048), (3, 4100), (2, 16384), (1030, 40)]


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,D", BN_SHAPES)
def test_block_norm(dev, types, rows, D):
    print(f"block_norm {rows}x{D} {types}", flush=True)
    x, y, gate, w_post, w_pre, a, gx, gz = _bn_inputs(rows, D, *types, dev)
    act = "silu" if D % 2 == 0 else "sigmoid"
    got = bn_run(x, y, gate, w_post, w_pre, a, 1e-6, act, gx, gz)
    assert got["x_new"].dtype == types[0] and got["z"].dtype == types[1]
    assert got["dx"].dtype == types[0] and got["dy"].dtype == got["dgate"].dtype == types[1]
    bn_check(got, bn_reference(x, y, gate, w_post, w_pre, a, 1e-6, act, gx, gz), rows)


# more rows than workgroups: each kernel variant carries its parameters' sums and the next row over
@pytest.mark.parametrize("types", [TYPES[0], TYPES[-1]], ids=[IDS[0], IDS[-1]])
@pytest.mark.parametrize("rows,D", [(5000, 96), (3200, 320), (1700, 1000), (800, 2040), (700, 999), (300, 4096),
                                    (300, 8184), (270, 16376), (260, 9001)])
def test_block_norm_many_rows(dev, types, rows, D):
    print(f"block_norm {rows}x{D} {types}", flush=True)
    x, y, gate, w_post, w_pre, a, gx, gz = _bn_inputs(rows, D, *types, dev, seed=2)
    got = bn_run(x, y, gate, w_post, w_pre, a, 1e-6, "silu", gx, gz)
    bn_check(got, bn_reference(x, y, gate, w_post, w_pre, a, 1e-6, "silu", gx, gz), rows)


@pytest.mark.parametrize("what", ["no_gate", "number", "only_x", "only_z", "large_eps"])
def test_block_norm_parts(dev, what):
    rows, D = 37, 192
    x, y, gate, w_post, w_pre, a, gx, gz = _bn_inputs(rows, D, torch.float32, torch.float32, dev, seed=1)
    eps = 0.5 if what == "large_eps" else 1e-6
    gate = None if what == "no_gate" else gate
    a = 0.75 if what == "number" else a
    gx, gz = None if what == "only_z" else gx, None if what == "only_x" else gz
    got = bn_run(x, y, gate, w_post, w_pre, a, eps, "silu", gx, gz)
    want = bn_reference(x, y, gate, w_post, w_pre, a, eps, "silu", gx, gz)
    bn_check({**got, "dw_pre": torch.zeros(D) if got["dw_pre"] is None else got["dw_pre"]}, want, rows)


def test_block_norm_rows_of_zeros_and_extremes(dev):
    """A row of zeros divides by sqrt(eps); rows near the type's ends stay finite where fp32 does."""
    from lifscan import hip_lm as LM
    D = 96
    x = torch.zeros(3, D, device=dev)
    y = torch.zeros(3, D, device=dev)
    y[1] = 1e15
    x[2] = -1e15
    w = torch.ones(D, device=dev)
    x_new, z = LM.block_norm(x, y, w, w)
    assert bool(torch.isfinite(x_new).all()) and bool(torch.isfinite(z).all())
    assert bool((z[0] == 0).all()) and float((x_new[1] - 1).abs().max()) < 1e-6
    assert float((z[2] + 1).abs().max()) < 1e-6
    x[0, 3] = float("nan")
    x_new, z = LM.block_norm(x, y, w, w)
    assert bool(torch.isnan(z[0]).all()) and bool(torch.isfinite(z[1:]).all())


def test_block_norm_against_differences(dev):
    """Central differences of the 64-bit sum of fp32 outputs along random directions: the step h leaves
    h^2 of the third derivative, of order one here, and the outputs' rounding over h."""
    from lifscan import hip_lm as LM
    rows, D, h = 6, 128, 2.0 ** -7
    x, y, gate, w_post, w_pre, a, gx, gz = _bn_inputs(rows, D, torch.float32, torch.float32, dev, seed=2)
    ops = [x, y, gate, w_post, w_pre, a]
    got = bn_run(*ops, 1e-6, "silu", gx, gz)

    def loss(ops):
        x_new, z = LM.block_norm(*ops[:2], ops[3], ops[4], gate=ops[2], res_scale=ops[5])
        return float((x_new.double() * gx).sum() + (z.double() * gz).sum())

    for i, k in enumerate(("dx", "dy", "dgate", "dw_post", "dw_pre", "da")):
        d = torch.randn(ops[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate(ops)] for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * h)
        want = float((got[k].double() * d).sum())
        assert abs(slope - want) <= 64 * h * h * float(got[k].double().norm()) * math.sqrt(2 * math.log(100)) \
            + 8 * F / h * float((got["x_new"].detach().double() * gx).norm() + (got["z"].detach().double() * gz).norm())


def test_block_norm_layouts_streams_and_bits(dev):
    from lifscan import hip_lm as LM
    x, y, gate, w_post, w_pre, a, gx, gz = _bn_inputs(60, 129, torch.float32, torch.bfloat16, dev, seed=3)
    want = bn_run(x, y, gate, w_post, w_pre, a, 1e-6, "silu", gx, gz)
    # [T, B, D] views in another order, an offset that no wide access takes, half-precision weights' cast
    turn = lambda t: t.view(6, 10, 129).transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bn_run(*(turn(t) for t in (x, y, gate)), w_post, w_pre, a, 1e-6, "silu", turn(gx), turn(gz))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k, t in got.items():
        assert torch.equal(t.reshape(want[k].shape), want[k]), k
    odd = [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(60, 129) for t in (x, y, gate)]
    x_new, z = LM.block_norm(*odd[:2], w_post, w_pre, gate=odd[2], res_scale=a)
    assert torch.equal(x_new, want["x_new"]) and torch.equal(z, want["z"])
    x_new, z = LM.block_norm(x[:0], y[:0], w_post, w_pre)
    assert x_new.shape == (0, 129) and z.dtype == torch.bfloat16
    empty = bn_run(x[:0], y[:0], gate[:0], w_post, w_pre, a, 1e-6, "silu", gx[:0], gz[:0])
    assert bool((empty["dw_post"] == 0).all()) and bool((empty["da"] == 0).all())
    for t in (torch.bfloat16, torch.float16):
        w = w_post.to(t).requires_grad_(True)
        LM.block_norm(x, y, w, w_pre)[0].sum().backward()
        assert w.grad.dtype == t


def test_block_norm_refusals(dev):
    from lifscan import hip_lm as LM
    x, w = torch.randn(4, 8, device=dev), torch.ones(8, device=dev)
    for f in (lambda: LM.block_norm(x.cpu(), x.cpu(), w.cpu(), w.cpu()), lambda: LM.block_norm(x, x[:2], w, w),
              lambda: LM.block_norm(x.half(), x, w, w), lambda: LM.block_norm(x.double(), x.double(), w, w),
              lambda: LM.block_norm(x, x, w[:4], w), lambda: LM.block_norm(x, x, w, w, gate=x.half()),
              lambda: LM.block_norm(x, x, w, w, gate=x, act="tanh"), lambda: LM.block_norm(x, x, w, w, eps=-1.0),
              lambda: LM.block_norm(x, x, w, w, res_scale=w[:3]),
              lambda: LM.block_norm(torch.randn(1, 16385, device=dev), torch.randn(1, 16385, device=dev),
                                    torch.ones(16385, device=dev), torch.ones(16385, device=dev))):
        with pytest.raises(ValueError):
            f()


# ----------------------------------------------------------------------------- embedding
def _tokens(n, V, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g)
    if kind == "one":
        return torch.full((n,), V // 2, dtype=torch.int64)
    if kind == "ordered":
        return torch.arange(n) % V
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return (torch.exp(u * math.log(V + 1)).long() - 1).clamp(0, V - 1)


EMBED_SHAPES = [(1, 1, 1), (5, 3, 9), (64, 1000, 64), (1000, 37, 257), (4097, 513, 130), (300, 70000, 24),
                (20000, 300, 16), (2, 5, 5000), (3000, 40000, 8)]


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["zipf", "uniform", "one", "ordered"])
@pytest.mark.parametrize("n,V,D", EMBED_SHAPES)
def test_embed(dev, dtype, kind, n, V, D):
    from lifscan import hip_lm as LM
    print(f"embed {n} {V} {D} {kind} {dtype}", flush=True)
    g = torch.Generator().manual_seed(n)
    tok = _tokens(n, V, kind, n)
    pad = int(tok[0]) if n > 3 and kind == "uniform" else None
    W = torch.randn(V, D, generator=g).to(dtype)
    dout = torch.randn(n, D, generator=g).to(dtype)
    Wg = W.to(dev).requires_grad_(True)
    out = LM.embed(tok.to(dev), Wg, scale=1.5, padding_idx=pad)
    (dW,) = torch.autograd.grad(out, Wg, dout.to(dev))
    keep = torch.ones(n, 1, dtype=torch.float64) if pad is None else (tok != pad).double()[:, None]
    close(out, 1.5 * W.double()[tok] * keep, 0.0)
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, tok, 1.5 * dout.double() * keep)
    size = torch.zeros(V, D, dtype=torch.float64).index_add_(0, tok, 1.5 * dout.double().abs() * keep)
    count = torch.bincount(tok, minlength=V).double()[:, None]
    assert dW.dtype == dtype
    close(dW, want, size * (2 + count), n=1)
    again = torch.autograd.grad(LM.embed(tok.to(dev), Wg, scale=1.5, padding_idx=pad), Wg, dout.to(dev))[0]
    assert torch.equal(dW, again)


@pytest.mark.parametrize("kind", ["zipf", "one"])
def test_embed_many_tokens_of_a_large_table(dev, kind):
    """More rows a workgroup than its waves can count apart, and more positions than its list holds."""
    test_embed(dev, torch.float32, kind, 6000, 200000, 8)


@pytest.mark.parametrize("kind", ["zipf", "uniform", "one", "ordered"])
@pytest.mark.parametrize("n,V,D", [(16385, 1, 1), (40000, 5, 3), (33333, 32000, 4), (70001, 200000, 2)])
def test_embed_many_tokens(dev, kind, n, V, D):
    """More tokens than one kernel sorts: split over the workgroups, with tables of few and of many rows."""
    test_embed(dev, torch.bfloat16 if kind == "zipf" else torch.float32, kind, n, V, D)


def test_embed_ids_outside_the_table(dev):
    """Ids below 0 and from V on read as zero rows and leave no gradient; also those that 32 bits fold."""
    from lifscan import hip_lm as LM
    W = torch.randn(10, 6, device=dev, requires_grad=True)
    tok = torch.tensor([[3, -1, 10], [2 ** 32 + 3, 9, -2 ** 31]], device=dev)
    out = LM.embed(tok, W)
    assert out.shape == (2, 3, 6)
    good = torch.zeros(2, 3, dtype=torch.bool)
    good[0, 0] = good[1, 1] = True
    assert torch.equal(out[0, 0], W[3]) and torch.equal(out[1, 1], W[9])
    assert bool((out[~good.to(dev)] == 0).all())
    (dW,) = torch.autograd.grad(out, W, torch.ones_like(out))
    want = torch.zeros(10, 6, device=dev)
    want[3] = want[9] = 1
    assert torch.equal(dW, want)


def test_embed_types_layouts_and_empty(dev):
    from lifscan import hip_lm as LM
    W = torch.randn(50, 33, device=dev)
    tok = _tokens(200, 50, "zipf").to(dev)
    want = LM.embed(tok, W)
    assert torch.equal(LM.embed(tok.int(), W), want)
    assert torch.equal(LM.embed(tok.view(20, 10).t(), W), want.view(20, 10, 33).transpose(0, 1))
    assert torch.equal(LM.embed(tok, W.t().contiguous().t()), want)
    shifted = torch.cat([W.flatten()[:1], W.flatten()])[1:].view(50, 33)
    assert torch.equal(LM.embed(tok, shifted), want)
    none = LM.embed(tok[:0], W.clone().requires_grad_(True))
    assert none.shape == (0, 33)
    Wg = W.clone().requires_grad_(True)
    (dW,) = torch.autograd.grad(LM.embed(tok[:0], Wg), Wg, none.detach())
    assert bool((dW == 0).all())
    # a gradient that is one row for every token
    (dW,) = torch.autograd.grad(LM.embed(tok, Wg).sum(), Wg)
    assert torch.equal(dW, torch.bincount(tok, minlength=50).float()[:, None].expand(50, 33))


def test_embed_gradient_against_differences(dev):
    """The lookup is linear: a whole step along the table changes <out, dout> by <dW, step>."""
    from lifscan import hip_lm as LM
    g = torch.Generator().manual_seed(4)
    tok = _tokens(500, 60, "zipf").to(dev)
    W, step = torch.randn(60, 40, generator=g).to(dev), torch.randn(60, 40, generator=g).to(dev)
    dout = torch.randn(500, 40, generator=g).to(dev)
    Wg = W.clone().requires_grad_(True)
    out = LM.embed(tok, Wg, scale=3.0)
    (dW,) = torch.autograd.grad(out, Wg, dout)
    moved = LM.embed(tok, W + step, scale=3.0)
    d = ((W + step).double() - W.double())
    change = float(((moved.double() - out.detach().double()) * dout.double()).sum())
    # roundings of the outputs and of sums of up to 500 rows
    tol = F * float(((moved.double().abs() + out.detach().double().abs()) * dout.double().abs()).sum())
    tol += 502 * F * float((torch.zeros_like(d).index_add_(0, tok, 3 * dout.double().abs()) * d.abs()).sum())
    assert abs(change - float((dW.double() * d).sum())) <= tol


def test_embed_refusals(dev):
    from lifscan import hip_lm as LM
    W, tok = torch.randn(5, 4, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for f in (lambda: LM.embed(tok.cpu(), W), lambda: LM.embed(tok, W.cpu()), lambda: LM.embed(tok.float(), W),
              lambda: LM.embed(tok, W[0]), lambda: LM.embed(tok, W.double()), lambda: LM.embed(tok, W, padding_idx=5),
              lambda: LM.embed(tok, W, padding_idx=-1), lambda: LM.embed(tok, W[:, :0])):
        with pytest.raises(ValueError):
            f()


# ----------------------------------------------------------------------------- distillation
def distill_reference(z, t, idx, tau, g):
    """(loss, dz, the sum of |terms| of each loss) in 64 bits."""
    z, t, g = z.detach().double().cpu() / tau, t.double().cpu() / tau, g.double().cpu()
    idx = idx.cpu()
    V = z.shape[1]
    there = (idx >= 0) & (idx < V)
    t = torch.where(there, t, -math.inf)
    some = (t > -math.inf).any(1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, t, 0.0), 1), 0.0)
    at = idx.clamp(0, V - 1)
    lse = torch.logsumexp(z, 1, keepdim=True)
    logq = torch.gather(z, 1, at) - lse
    terms = torch.where(p > 0, p * (torch.log(p.clamp(min=1e-300)) - logq), 0.0)
    size = torch.where(p > 0, p * (torch.log(p.clamp(min=1e-300)).abs() + torch.gather(z, 1, at).abs() + lse.abs()), 0.0)
    q = torch.exp(z - lse)
    dz = torch.where(some, q, 0.0).scatter_add(1, at, -p) * (g * tau)[:, None]
    return tau * tau * terms.sum(1), dz, tau * tau * size.sum(1), (q.abs() + 1) * (g.abs() * tau)[:, None]


def _distill_inputs(rows, V, K, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed + V)
    z = (3 * torch.randn(rows, V, generator=g)).to(dtype)
    noisy = z.float() + torch.randn(rows, V, generator=g)
    top = noisy.topk(min(K, V), 1)
    idx = top.indices.clone()
    if idx.shape[1]:
        cut = torch.randint(0, idx.shape[1] + 1, (rows, 1), generator=g)
        idx[torch.arange(idx.shape[1]) >= cut] = -1
    return z.to(dev), top.values.to(dtype).to(dev), idx.to(dev), torch.randn(rows, generator=g).to(dev)


def distill_check(z, t, idx, tau, g, V):
    from lifscan import hip_lm as LM
    zg = z.detach().requires_grad_(True)
    loss = LM.distill_topk(zg, t, idx, temperature=tau)
    (dz,) = torch.autograd.grad(loss, zg, g)
    want, dwant, size, dsize = distill_reference(z, t, idx, tau, g)
    assert loss.dtype == torch.float32 and dz.dtype == z.dtype
    # exp of an argument off by |z| 2^-24: the probabilities' relative error
    most = 64 + 2 * float(z.detach().abs().max()) / tau
    close(loss, want, size + tau * tau, n=most)
    # below its normal range a 16-bit type has absolute steps
    bound = U[dz.dtype] * dwant.abs() + most * F * dsize.clamp(max=1e300)
    bound += 2.0 ** -25 if dz.dtype == torch.float16 else 0.0
    err = (dz.double().cpu() - dwant).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return loss, dz


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V,K,tau", [(1, 1, 1, 1.0), (3, 7, 7, 2.0), (5, 1000, 16, 1.0), (40, 257, 64, 3.5),
                                          (2, 70001, 100, 2.0), (1, 131072, 5, 1.0), (300, 515, 1, 0.5),
                                          (7, 4096, 1024, 1.5), (600, 32, 8, 2.0)])
def test_distill(dev, dtype, rows, V, K, tau):
    print(f"distill {rows}x{V} K={K} {dtype}", flush=True)
    z, t, idx, g = _distill_inputs(rows, V, K, dtype, dev)
    loss, dz = distill_check(z, t, idx, tau, g, V)
    assert bool((loss[(idx < 0).all(1)] == 0).all()) and bool((dz[(idx < 0).all(1)] == 0).all())


@pytest.mark.parametrize("rows,V,K", [(520, 40000, 384), (2, 70001, 4096)])
def test_distill_many_entries(dev, rows, V, K):
    """Ids that lie 32768 apart, and ids that are named two to four times, among many."""
    print(f"distill {rows}x{V} K={K}", flush=True)
    gen = torch.Generator().manual_seed(V)
    z = 3 * torch.randn(rows, V, generator=gen)
    low = torch.rand(rows, V - 32768, generator=gen).topk(K // 3, 1).indices
    idx = torch.cat([low, low + 32768, torch.randint(0, V, (rows, K - 2 * (K // 3) - 6), generator=gen),
                     low[:, :3], low[:, :3]], 1)
    idx = idx[:, torch.randperm(K, generator=gen)].contiguous()
    t = torch.gather(z, 1, idx) + torch.randn(rows, K, generator=gen)
    distill_check(z.to(dev), t.to(dev), idx.to(dev), 1.5, torch.randn(rows, generator=gen).to(dev), V)


def test_distill_entries(dev):
    """No entry at all, K = 0, ids beyond the vocabulary, one id named twice, teacher logits of -inf, fp32
    teacher values with bf16 logits, logits of -inf that the teacher does not name."""
    from lifscan import hip_lm as LM
    V = 700
    for dtype in U:
        z, t, idx, g = _distill_inputs(6, V, 8, dtype, dev, seed=5)
        idx[0] = -1
        idx[1] = torch.tensor([5, 5, 9, 5, -1, V, 2 ** 32 + 4, -7])
        idx[2] = torch.arange(8)
        t[2, :7] = float("-inf")
        idx[3] = torch.arange(10, 18)
        z[3, 100:600] = float("-inf")
        t[3] = t[3].float()
        distill_check(z, t, idx, 2.0, g, V)
        distill_check(z, t.float() + 1e-4, idx, 2.0, g, V)
        t[2] = float("-inf")  # a row whose teacher has no weight anywhere
        zg = z.clone().requires_grad_(True)
        loss = LM.distill_topk(zg, t, idx, temperature=2.0)
        assert bool((loss[[0, 2]] == 0).all())
        (dz,) = torch.autograd.grad(loss, zg, g)
        assert bool((dz[0] == 0).all()) and bool((dz[2] == 0).all()) and bool((dz[3, 100:600] == 0).all())
    loss = LM.distill_topk(z, t[:, :0], idx[:, :0])
    assert loss.shape == (6,) and bool((loss == 0).all())
    # a named id that the student rules out costs infinitely much
    z = torch.zeros(1, 5, device=dev)
    z[0, 2] = float("-inf")
    loss = LM.distill_topk(z, torch.zeros(1, 2, device=dev), torch.tensor([[2, 3]], device=dev))
    assert float(loss) == float("inf")
    # a NaN logit is the row's own matter
    z = torch.zeros(2, 300, device=dev)
    z[0, 7] = float("nan")
    loss = LM.distill_topk(z, torch.zeros(2, 1, device=dev), torch.tensor([[1], [1]], device=dev))
    assert math.isnan(float(loss[0])) and abs(float(loss[1]) - math.log(300)) < 1e-5


def test_distill_large_logits_do_not_overflow(dev):
    z = torch.zeros(2, 400, device=dev)
    z[0, 3], z[1] = 3e4, -3e4
    z[1, 8] = 3e4
    idx = torch.tensor([[3, 4], [9, 8]], device=dev)
    distill_check(z, torch.tensor([[3e4, 0.0], [-3e4, 3e4]], device=dev), idx, 1.0, torch.ones(2, device=dev), 400)


def test_distill_against_differences(dev):
    from lifscan import hip_lm as LM
    rows, V, tau, h = 4, 50, 2.0, 2.0 ** -6
    z, t, idx, g = _distill_inputs(rows, V, 8, torch.float32, dev, seed=6)
    zg = z.clone().requires_grad_(True)
    (dz,) = torch.autograd.grad(LM.distill_topk(zg, t, idx, temperature=tau), zg, g)
    d = torch.randn(rows, V, generator=torch.Generator().manual_seed(1)).to(dev)
    up, down = (LM.distill_topk(z + s * h * d, t, idx, temperature=tau).double() for s in (1, -1))
    slope = float(((up - down) * g).sum()) / (2 * h)
    # h^2/6 of the third derivative along d (below |d|_inf^3 / tau of order ten), rounding of the losses over h
    tol = h * h / 6 * 64 * float(g.abs().sum()) + 64 * F / h * float((up.abs() * g.abs()).sum() + g.abs().sum() * 16)
    assert abs(slope - float((dz.double() * d).sum())) <= tol


def test_distill_layouts_streams_and_bits(dev):
    from lifscan import hip_lm as LM
    z, t, idx, g = _distill_inputs(24, 1003, 16, torch.bfloat16, dev, seed=7)
    zg = z.clone().requires_grad_(True)
    loss = LM.distill_topk(zg, t, idx)
    (want,) = torch.autograd.grad(loss, zg, g)
    # rows of a wider array, [T, B, V] arrays, a broadcast gradient, another stream
    wide = torch.randn(24, 1100, device=dev).to(torch.bfloat16)
    wide[:, 40:1043] = z
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        wg = wide.requires_grad_(True)
        got = LM.distill_topk(wg[:, 40:1043], t, idx)
        (dw,) = torch.autograd.grad(got, wg, g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, loss) and torch.equal(dw[:, 40:1043], want)
    cube = LM.distill_topk(z.view(4, 6, 1003), t.view(4, 6, 16), idx.view(4, 6, 16))
    assert torch.equal(cube.flatten(), loss)
    (d1,) = torch.autograd.grad(LM.distill_topk(zg, t, idx).sum(), zg)
    (d2,) = torch.autograd.grad(LM.distill_topk(zg, t, idx), zg, torch.ones(24, device=dev))
    assert torch.equal(d1, d2)
    none = LM.distill_topk(zg[:0], t[:0], idx[:0])
    assert none.shape == (0,)
    (d0,) = torch.autograd.grad(none, zg, none.detach())
    assert bool((d0 == 0).all())


def test_distill_refusals(dev):
    from lifscan import hip_lm as LM
    z, t, idx = torch.randn(2, 9, device=dev), torch.randn(2, 3, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev)
    for f in (lambda: LM.distill_topk(z.cpu(), t, idx), lambda: LM.distill_topk(z, t.cpu(), idx),
              lambda: LM.distill_topk(z.double(), t, idx), lambda: LM.distill_topk(z, t[:1], idx),
              lambda: LM.distill_topk(z, t, idx[:, :2]), lambda: LM.distill_topk(z, t, idx.int()),
              lambda: LM.distill_topk(z, idx, idx), lambda: LM.distill_topk(z, t, idx, temperature=0.0),
              lambda: LM.distill_topk(z, t, idx, temperature=float("inf")),
              lambda: LM.distill_topk(z, torch.randn(2, 4097, device=dev), torch.zeros(2, 4097, dtype=torch.int64, device=dev))):
        with pytest.raises(ValueError):
            f()


def test_row_operators_in_a_graph(dev):
    """Lookup, norms and loss with their gradients, captured and replayed three times."""
    from lifscan import hip_lm as LM
    W = torch.randn(500, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    tok = _tokens(96, 500, "zipf").to(dev)
    _, t, idx, _ = _distill_inputs(96, 64, 8, torch.float32, dev)

    def work():
        e = LM.embed(tok, W, scale=2.0)
        x, z = LM.block_norm(e, e * 0.5, w, w, gate=e, res_scale=0.5)
        return torch.autograd.grad(LM.distill_topk(z, t, idx, temperature=2.0), (W, w),
                                   torch.ones(96, device=dev))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    want = [t.clone() for t in work()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        work()
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", list(U), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [300, 9001])
def test_distill_teacher_values_that_are_nan(dev, dtype, V):
    """A NaN among a row's teacher values is an entry, also where every other one is NaN or -inf: the row's loss
    is NaN, its gradient NaN at the entries' places, and other rows are as without it."""
    from lifscan import hip_lm as LM
    z, t, idx, g = _distill_inputs(5, V, 8, dtype, dev, seed=11)
    idx[:] = torch.arange(8, device=dev) * 7
    loss, dz = distill_check(z, t, idx, 2.0, g, V)
    bad = t.clone()
    bad[1] = float("nan")
    bad[2, 0] = float("nan")
    bad[3] = float("-inf")
    bad[3, 5] = float("nan")
    zg = z.clone().requires_grad_(True)
    got = LM.distill_topk(zg, bad, idx, temperature=2.0)
    (dbad,) = torch.autograd.grad(got, zg, g)
    assert got.isnan().tolist() == [False, True, True, True, False]
    for row in (0, 4):
        assert got[row] == loss[row].detach() and torch.equal(dbad[row], dz[row])
    for row in (1, 2, 3):
        assert bool(dbad[row, idx[row]].isnan().all())
        other = torch.ones(V, dtype=torch.bool, device=dev)
        other[idx[row]] = False
        assert bool(dbad[row, other].isfinite().all())


def test_forward_mode_and_traces_are_refused(dev):
    """A dual tensor's tangent would be lost, and a trace would record none of the kernels."""
    import torch.autograd.forward_ad as fw
    from lifscan import hip_linattn as LA
    from lifscan import hip_lm as LM
    x, w, q = torch.randn(4, 8, device=dev), torch.ones(8, device=dev), torch.randn(4, 1, 2, 8, device=dev)
    s, b = torch.zeros(1, 2, 8, 8, device=dev), torch.full((2,), 0.9, device=dev)
    tok = torch.zeros(3, dtype=torch.int64, device=dev)
    idx = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    calls = [
        (lambda *a: LA.lin_attn(*a)[0], (q, q, q, b, s)),
        (lambda *a: LA.lin_attn_step(*a), (q[0], q[0], q[0], b, s)),
        (lambda *a: LM.block_norm(*a)[0], (x, x, w, w, x, w)),
        (lambda a: LM.embed(tok, a), (x,)),
        (lambda a, v: LM.distill_topk(a, v, idx), (x, x[:, :2].contiguous())),
    ]
    for f, args in calls:
        f(*args)
        for i in range(len(args)):
            with fw.dual_level():
                duals = [fw.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*duals)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, args, check_trace=False)
        f(*args)


def test_gradients_that_arrive_in_other_forms(dev):
    """A dual gradient is refused in the backward too; a lazily negated one is read with its sign."""
    import torch.autograd.forward_ad as fw
    from lifscan import hip_linattn as LA
    from lifscan import hip_lm as LM
    x, q = torch.randn(4, 8, device=dev), torch.randn(4, 1, 2, 8, device=dev)
    w = torch.ones(8, device=dev)
    tok, idx = torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(4, 2, dtype=torch.int64, device=dev)
    for f, a in ((lambda a: LA.lin_attn(a, a, a, 0.9)[0], q), (lambda a: LM.block_norm(a, a, w, w)[1], x),
                 (lambda a: LM.embed(tok, a), x), (lambda a: LM.distill_topk(a, x[:, :2], idx), x)):
        a = a.clone().requires_grad_(True)
        out = f(a)
        g = torch.randn_like(out)
        (want,) = torch.autograd.grad(out, a, -g, retain_graph=True)
        (got,) = torch.autograd.grad(out, a, torch._neg_view(g), retain_graph=True)
        assert torch.equal(got, want)
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, a, fw.make_dual(g, g))
    for f in (lambda: LM.block_norm(torch._neg_view(x), x, w, w), lambda: LA.lin_attn(q, torch._neg_view(q), q, 0.9),
              lambda: LM.embed(tok, torch._neg_view(x)), lambda: LM.distill_topk(torch._neg_view(x), x[:, :2], idx)):
        with pytest.raises(ValueError):
            f()


def test_embed_padding_beyond_32_bits(dev):
    """A padding id that no token of the table has takes no row away, whatever its lower 32 bits."""
    from lifscan import _native as n
    L = n.lib()
    V, D = 10, 8
    tok = torch.tensor([3, 3, 5, 0], device=dev)
    W, dout = torch.randn(V, D, device=dev), torch.randn(4, D, device=dev)
    out, dW = torch.empty(4, D, device=dev), torch.empty(V, D, device=dev)
    nb = L.lsh_embed_bwd_workspace(4, V)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    st = n.stream_of(W)
    for pad in (2 ** 32 + 3, -(2 ** 32) + 5, 2 ** 32 - 1):
        assert L.lsh_embed_fwd(0, n.ptr(tok), n.ptr(W), n.ptr(out), 4, V, D, pad, 1.0, st) == 0
        assert L.lsh_embed_bwd(0, n.ptr(tok), n.ptr(dout), n.ptr(dW), 4, V, D, pad, 1.0, n.ptr(ws), nb, st) == 0
        assert torch.equal(out, W[tok])
        assert torch.equal(dW[3], dout[0] + dout[1]) and torch.equal(dW[5], dout[2]) and torch.equal(dW[0], dout[3])


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]], ids=[IDS[0], IDS[3]])
def test_block_norm_wide_gates(dev, types, act):
    """Gates far from zero: a sigmoid's derivative keeps its digits where the sigmoid is nearly one."""
    rows, D = 40, 512
    x, y, gate, w_post, w_pre, a, gx, gz = _bn_inputs(rows, D, *types, dev, seed=4)
    gate = torch.linspace(-30, 30, rows * D).view(D, rows).t().contiguous().to(types[1]).to(dev)
    got = bn_run(x, y, gate, w_post, w_pre, a, 1e-6, act, gx, gz)
    want = bn_reference(x, y, gate, w_post, w_pre, a, 1e-6, act, gx, gz)
    if act == "sigmoid":  # 1 - sg has lost its digits at 30 in 64 bits too: sigmoid(-gate) in its place
        g = gate.double().cpu()
        right = (1 / (1 + torch.exp(g))) / (1 - 1 / (1 + torch.exp(-g)))
        want["dgate"], want["size"]["dgate"] = want["dgate"] * right, want["size"]["dgate"] * right
    bn_check(got, want, rows)
