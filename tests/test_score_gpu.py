"""GPU: log probabilities of given tokens, entropy and alternatives (lifscan.hip_lm.token_logprobs) against
their definitions in 64 bits, the gradient against the written-out formula in 64 bits and against differences.

Tolerances.  F = 2^-24.  A difference (z - m)/tau in base 2 is off by 2 F of itself, so its power by some 2 F
of the difference; a thread adds up to V/256 terms one after the other, then some ten more levels.  So log
probabilities and entropies are off by (64 + V/64) F of 1 + |log p| + log(sum), the alternatives' ids not at
all, and a gradient by as much of p times the factors that it multiplies, each as an absolute value, and the
rounding to its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def inputs(rows, V, dtype, dev, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed + rows + 3 * V)
    z = (spread * torch.randn(rows, V, generator=g)).to(dtype)
    tok = torch.randint(-1, V + 1, (rows,), generator=g)  # some outside on either side
    return z.to(dev), tok.to(dev), torch.randn(rows, generator=g).to(dev), torch.randn(rows, generator=g).to(dev)


def reference(z, tok, tau, K, gl=None, gh=None):
    """64 bits on the CPU; rows of -inf alone: log p = -inf, entropy 0, no gradient."""
    z0, tok = z.detach().double().cpu(), tok.cpu().long()
    V = z0.shape[1]
    z = z0 / tau
    m = z.max(1, keepdim=True).values
    none = (m == -math.inf)
    e = torch.where(none, 0.0, torch.exp(z - m))
    l = torch.log(e.sum(1, keepdim=True))
    lp = torch.where(none, -math.inf, z - m - l)
    p = torch.exp(lp)
    H = -torch.special.xlogy(p, p).sum(1)
    there = (tok >= 0) & (tok < V)
    at = torch.where(there, tok, 0)[:, None]
    logp = torch.where(there, lp.gather(1, at)[:, 0], 0.0)
    out = {"logp": logp, "entropy": H, "l": torch.where(none, 0.0, l)[:, 0]}
    # a stable sort leaves equal values in the order of their ids; the two zeros are equal
    order = torch.sort(torch.where(z0 == 0, 0.0, z0), dim=1, descending=True, stable=True).indices[:, :K]
    out["index"], out["top"] = order, lp.gather(1, order)
    if gl is not None or gh is not None:
        gl = torch.zeros(len(tok)) if gl is None else gl.cpu()
        gh = torch.zeros(len(tok)) if gh is None else gh.cpu()
        gl, gh = torch.where(there, gl.double(), 0.0)[:, None], gh.double()[:, None]
        plp = torch.special.xlogy(p, p)
        d = -gl * p - gh * (plp + p * H[:, None])
        d.scatter_add_(1, at, gl)
        size = gl.abs() * p + gh.abs() * (plp.abs() + p * H[:, None])
        size = size * (1 + torch.where(p > 0, lp.abs(), 0.0) + out["l"][:, None])
        size.scatter_add_(1, at, gl.abs())
        keep = ~none
        out["dz"], out["size"] = torch.where(keep, d, 0.0) / tau, torch.where(keep, size, 0.0) / tau
    return out


def same(got, want, bound):
    got = got.detach().double().cpu()
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    err = (got - want).abs()[~inf]
    b = bound[~inf]
    assert bool((err <= b).all()), float((err / b).max())


def check(out, dz, want, V, K):
    n = (64 + V / 64) * F
    l = want["l"]
    same(out[0], want["logp"], n * (1 + want["logp"].abs() + l))
    same(out[1], want["entropy"], n * (1 + want["entropy"] + l))
    if K:
        assert out[3].dtype == torch.int64 and torch.equal(out[3].cpu(), want["index"])
        same(out[2], want["top"], n * (1 + want["top"].abs() + l[:, None]))
    if dz is not None:
        err = (dz.double().cpu() - want["dz"]).abs()
        bound = U[dz.dtype] * want["dz"].abs() + n * want["size"] + (2.0 ** -25 if dz.dtype == torch.float16 else 2.0 ** -126)
        assert bool((err <= bound).all()), float((err / bound).max())


def run(z, tok, tau, K, gl=None, gh=None):
    from lifscan import hip_lm as LM
    zg = z.detach().requires_grad_(True)
    out = LM.token_logprobs(zg, tok, temperature=tau, top=K)
    outs = [(o, g) for o, g in ((out[0], gl), (out[1], gh)) if g is not None]
    (dz,) = torch.autograd.grad([o for o, _ in outs], zg, [g for _, g in outs])
    return out, dz


SHAPES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 64, 64), (4, 100, 20), (3, 257, 1), (2, 2047, 5), (3, 2048, 64), (2, 4097, 20),
          (3, 8192, 5), (2, 8200, 64), (2, 9001, 20), (1, 40003, 64), (40, 33000, 20), (1500, 130, 7), (1100, 8209, 20)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,V,K", SHAPES)
def test_values_and_gradients(dev, dtype, rows, V, K):
    print(f"score {rows}x{V} top {K} {dtype}", flush=True)
    tau = (1.0, 0.7, 2.0)[V % 3]
    z, tok, gl, gh = inputs(rows, V, dtype, dev)
    out, dz = run(z, tok, tau, K, gl, gh)
    assert dz.dtype == dtype and out[0].dtype == out[1].dtype == torch.float32
    check(out, dz, reference(z, tok, tau, K, gl, gh), V, K)


@pytest.mark.parametrize("which", ["logp", "entropy"])
def test_parts_of_the_gradient(dev, which):
    z, tok, gl, gh = inputs(9, 1000, torch.float32, dev, seed=1)
    gl, gh = (gl, None) if which == "logp" else (None, gh)
    out, dz = run(z, tok, 1.3, 0, gl, gh)
    assert len(out) == 2
    check(out, dz, reference(z, tok, 1.3, 0, gl, gh), 1000, 0)


def test_sums_send_expanded_gradients(dev):
    from lifscan import hip_lm as LM
    z, tok, *_ = inputs(9, 1000, torch.float32, dev, seed=2)
    zg = z.clone().requires_grad_(True)
    logp, H = LM.token_logprobs(zg, tok)
    (logp.sum() * 0.5 + H.mean()).backward()
    one = torch.ones(9, device=dev)
    want = reference(z, tok, 1.0, 0, 0.5 * one, one / 9)
    check((logp, H), zg.grad, want, 1000, 0)


# what few threads hold between them, runs of equal values, and masks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 9001, 33000])
@pytest.mark.parametrize("rows", [2, 1200])
def test_alternatives_in_any_order(dev, dtype, V, rows):
    from lifscan import hip_lm as LM
    if rows > 2 and V > 9001:
        V = 20011
    K = 64
    i = torch.arange(V)
    made = {
        "rising": i.double() / V * 8, "falling": -i.double() / V * 8, "equal": torch.zeros(V).double(),
        "zeros of both signs": torch.where(i % 3 == 0, -0.0, 0.0).double(),
        # the largest in a few threads' share: pieces of 8 (or 4) elements every 256
        "one thread in a row": torch.where((i // 8) % 256 < 2, 5.0 + i.double() / V, -1.0 - i.double() / V),
        "one piece": torch.where(i < 40, 3.0, 1.0).double(),
        "nearly all masked": torch.where(i % 1000 == 7, i.double() / V, -math.inf),
        "all masked": torch.full((V,), -math.inf).double(),
        "last": torch.where(i == V - 1, 9.0, 0.0).double(),
    }
    for name, row in made.items():
        print(f"alternatives {rows}x{V} {dtype}: {name}", flush=True)
        z = row.to(dtype).to(dev).expand(rows, V).contiguous()
        tok = torch.arange(rows, device=dev) * 7 % V
        gl, gh = torch.ones(rows, device=dev), torch.ones(rows, device=dev)
        out, dz = run(z, tok, 1.0, K, gl, gh)
        few = slice(0, 2)
        want = reference(z[few], tok[few], 1.0, K, gl[few], gh[few])
        check([o[few] for o in out], dz[few], want, V, K)
        assert torch.equal(out[3], out[3][:1].expand(rows, K)), name
        if name == "all masked":
            assert bool((out[1] == 0).all()) and bool((out[0] == -math.inf).all()) and not bool(dz.any())


@pytest.mark.parametrize("K", [1, 5, 20])
@pytest.mark.parametrize("rows,V", [(8, 1001), (1104, 300), (1104, 20011), (8, 70001)])
def test_few_alternatives_of_long_runs(dev, rows, V, K):
    """More threads reach the bound than alternatives are asked for: equal values behind, between and before larger ones."""
    from lifscan import hip_lm as LM
    g = torch.Generator().manual_seed(V + K)
    i = torch.arange(V)
    for dtype in (torch.float32, torch.float16):
        for low in (-math.inf, torch.finfo(dtype).min, 0.0, -0.0, 2.5):
            print(f"alternatives of runs {rows}x{V} top {K} {dtype}: {low}", flush=True)
            z = torch.full((8, V), low)
            z[1, torch.randperm(V, generator=g)[:K // 2]] = 3.0  # fewer larger ones than alternatives
            z[2, V // 2:] = 4.0
            z[3, :V // 3] = 4.0
            z[4] = torch.where(i % 3 == 1, 3.0, z[4])
            z[5] = torch.where(i >= V - 2, 5.0, torch.where(i % 7 == 3, 3.0, z[5]))
            z[6] = torch.where(i % 777 == 5, 3.0 + (i % 5), z[6])
            z[7] = torch.where((i // 64) % 9 == 8, 3.0, -7.0)
            z = z.to(dtype)
            want = reference(z, torch.zeros(8, dtype=torch.int64), 1.0, K)
            out = LM.token_logprobs(z.to(dev).repeat(rows // 8, 1), torch.zeros(rows, dtype=torch.int64, device=dev), top=K)
            check([o[:8] for o in out], None, want, V, K)
            assert torch.equal(out[3], out[3][:8].repeat(rows // 8, 1))


@pytest.mark.parametrize("V", [500, 9000, 70000])
def test_many_large_values_in_few_threads(dev, V):
    """More values reach the bound than the list holds: 60 pieces' threads hold the largest of every block."""
    from lifscan import hip_lm as LM
    for rows in (1, 1100 if V <= 9000 else 2):
        i = torch.arange(V)
        z = torch.where((i // 4) % 256 < 30, 5.0 + (i * 37 % V).double() / V, -3.0 - i.double() / V).float()
        z = z.to(dev).expand(rows, V).contiguous()
        tok = torch.zeros(rows, dtype=torch.int64, device=dev)
        out = LM.token_logprobs(z, tok, top=64)
        want = reference(z[:1], tok[:1], 1.0, 64)
        check([o[:1] for o in out], None, want, V, 64)
        assert torch.equal(out[3], out[3][:1].expand(rows, 64))


@pytest.mark.parametrize("V", [50, 9001])
def test_values_that_are_not_finite(dev, V):
    """NaN and +inf make their row's results NaN and no other's; NaN comes first among the alternatives, then
    +inf; masked logits count for nothing."""
    rows, K = 6, 5
    z, tok, gl, gh = inputs(rows, V, torch.float32, dev, seed=3)
    tok.clamp_(0, 20)
    want, dwant = run(z, tok, 1.0, K, gl, gh)
    bad = z.clone()
    bad[1, 30] = float("nan")
    bad[2, 31] = float("inf")
    bad[3] = float("nan")
    bad[4, 25:] = -math.inf
    got, dz = run(bad, tok, 1.0, K, gl, gh)
    for r in (0, 5):
        for a, b in zip(got, want):
            assert torch.equal(a[r], b[r])
        assert torch.equal(dz[r], dwant[r])
    for r in (1, 2, 3):
        assert bool(got[0][r].isnan()) and bool(got[1][r].isnan()) and bool(dz[r].isnan().any())
    assert int(got[3][1, 0]) == 30 and int(got[3][2, 0]) == 31 and got[3][3].tolist() == list(range(K))
    ref = reference(bad[4:5], tok[4:5], 1.0, K, gl[4:5], gh[4:5])
    check([o[4:5] for o in got], dz[4:5], ref, V, K)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("V", [40, 9001])
def test_masks_of_the_lowest_value(dev, dtype, V):
    """Logits at the lowest value of their type are values: far below the others they have probability 0, and a
    row of nothing else is uniform.  Such a difference times 1/tau is no fp32 number: it is not to become NaN."""
    low = torch.finfo(dtype).min
    z, tok, gl, gh = inputs(4, V, dtype, dev, seed=17)
    tok = torch.tensor([3, 3, 5, 7], device=dev)
    z[0, 6:] = low
    z[1, :] = low
    z[2, 5] = low
    z[3, 7] = torch.finfo(dtype).max
    out, dz = run(z, tok, 0.7, 5, gl, gh)
    if dtype == torch.float16:
        check(out, dz, reference(z, tok, 0.7, 5, gl, gh), V, 5)
    else:  # 3.4e38 / 0.7 is beyond fp32, the type of the results: rounded, it is infinite
        assert float(out[0][2]) == -math.inf
    assert bool(dz.isfinite().all()) and not bool(torch.stack(out[:2]).isnan().any()) and not bool(out[2].isnan().any())
    assert float((out[0][1] + math.log(V)).abs()) < 1e-5 and float((out[1][1] - math.log(V)).abs()) < 1e-5
    assert out[3][1].tolist() == [0, 1, 2, 3, 4] and int(out[3][3, 0]) == 7 and float(out[1][3]) < 1e-5
    want = reference(z[:1, :6], tok[:1], 0.7, 5, gl[:1], gh[:1])
    check([o[:1] for o in out], dz[:1, :6], want, V, 5)
    assert not bool(dz[0, 6:].any())


@pytest.mark.parametrize("tau", [1.0, 2.0])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,V", [(3, 40), (3, 9001), (3, 70001), (1104, 9001)])
def test_log_probabilities_of_the_lowest_value(dev, dtype, rows, V, tau):
    """They are fp32 numbers, also where the logit's distance from the largest in other units, or before it is divided, is
    none."""
    z, _, gl, gh = inputs(3, V, dtype, dev, seed=19)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z[:, 5:] = low
    z[1, 2] = -low if tau > 1 else 8.0
    z[2, :] = low
    z[2, V - 1] = high / 2 if tau > 1 else 3.0
    tok = torch.tensor([6, V - 1, 0], device=dev)
    out, dz = run(z.repeat(rows // 3, 1), tok.repeat(rows // 3), tau, 20, gl.repeat(rows // 3), gh.repeat(rows // 3))
    want = reference(z, tok, tau, 20, gl, gh)
    assert bool(want["logp"].float().isfinite().all()) and bool((want["logp"] < -1e4).all())
    check([o[:3] for o in out], dz[:3], want, V, 20)
    assert all(torch.equal(o, o[:3].repeat((rows // 3,) + (1,) * (o.dim() - 1))) for o in out)


@pytest.mark.parametrize("tau", [0.7, 1.0])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,V", [(6, 40), (6, 9001), (6, 70001), (1104, 9001)])
def test_masks_of_both_kinds(dev, dtype, rows, V, tau):
    """-inf beside the lowest value of the type and nothing larger: log p is -inf there and uniform over the others, also
    where the lowest value over tau is no fp32 number.  A row with NaN or +inf has NaN."""
    low = torch.finfo(dtype).min
    z, _, gl, gh = inputs(6, V, dtype, dev, seed=23)
    i = torch.arange(V, device=dev)
    z[0] = torch.where(i < 6, low, -math.inf)
    z[1] = torch.where(i == V - 1, -math.inf, low)
    z[2] = torch.where(i % 3 == 1, low, -math.inf)
    z[3] = torch.where(i == V // 2, low, -math.inf)
    z[4] = torch.where(i == 9, math.nan, z[0].float()).to(dtype)
    z[5] = torch.where(i == 9, math.inf, z[0].float()).to(dtype)
    tok = torch.tensor([7, V - 1, 1, 2, 7, 7], device=dev)
    n = rows // 6
    out, dz = run(z.repeat(n, 1), tok.repeat(n), tau, 20, gl.repeat(n), gh.repeat(n))
    want = reference(z[:4], tok[:4], tau, 20, gl[:4], gh[:4])
    assert want["logp"].isinf().tolist() == [True, True, False, True] and int(want["top"].isinf().sum()) == 14 + 19 + (7 if V == 40 else 0)
    check([o[:4] for o in out], dz[:4], want, V, 20)
    for o in out[:3]:
        assert bool(o[4:6].isnan().all())
    for o in out:
        assert bool(((o == o[:6].repeat((n,) + (1,) * (o.dim() - 1))) | o.isnan()).all())



def test_tokens_outside_the_vocabulary(dev):
    from lifscan import hip_lm as LM
    z, _, gl, gh = inputs(6, 77, torch.float32, dev, seed=4)
    tok = torch.tensor([-1, 77, -100, 2 ** 40, -2 ** 40, 76], device=dev)
    out, dz = run(z, tok, 1.0, 0, gl, gh)
    check(out, dz, reference(z, tok, 1.0, 0, gl, gh), 77, 0)
    assert not bool(out[0][:5].any()) and float(out[0][5]) < 0
    (d,) = torch.autograd.grad(LM.token_logprobs(y := z.clone().requires_grad_(True), tok)[0].sum(), y)
    assert not bool(d[:5].any()) and bool(d[5].any())
    a, b = LM.token_logprobs(z, tok.clamp(-1, 77).int()), LM.token_logprobs(z, tok)
    assert torch.equal(a[0], b[0])


def test_large_logits_and_temperatures(dev):
    z, tok, gl, gh = inputs(4, 3000, torch.float32, dev, seed=5, spread=1.0)
    tok.clamp_(0, 2999)
    for scale, tau in ((1e4, 1.0), (1.0, 1e-3), (3e37, 1e36), (1.0, 1e3)):
        out, dz = run(z * scale, tok, tau, 3, gl, gh)
        want = reference(z * scale, tok, tau, 3, gl, gh)
        # differences of thousands: their own rounding, 4 F of them, is what counts
        n = (64 + 3000 / 64) * F
        same(out[0], want["logp"], n * (1 + want["logp"].abs() + want["l"]))
        same(out[1], want["entropy"], n * (1 + want["entropy"] + want["l"]))
        assert torch.equal(out[3].cpu(), want["index"]) and bool(dz.isfinite().all())


def test_gradient_against_differences(dev):
    """Central differences of the outputs' 64-bit sum with steps of 2^-5 (the third derivative leaves some
    2^-10 of the terms' sum), in a vocabulary whose outputs are of size 10: their roundings 10 * 2^-24 * 2^5."""
    from lifscan import hip_lm as LM
    z, tok, gl, gh = inputs(5, 300, torch.float32, dev, seed=6)
    _, dz = run(z, tok, 0.8, 0, gl, gh)

    def value(z):
        a, b = LM.token_logprobs(z, tok, temperature=0.8)
        return float((a.double() * gl.double()).sum() + (b.double() * gh.double()).sum())

    for n in range(4):
        v = torch.randn(z.shape, generator=torch.Generator().manual_seed(n)).to(dev)
        step = 2.0 ** -5
        diff = (value(z + step * v) - value(z - step * v)) / (2 * step)
        want = float((dz.double() * v.double()).sum())
        assert abs(diff - want) <= 2.0 ** -9 * float((dz.double() * v.double()).abs().sum()) + 2.0 ** -12


def test_layouts_streams_and_bits(dev):
    from lifscan import hip_lm as LM
    z, tok, gl, gh = inputs(6, 999, torch.bfloat16, dev, seed=7)
    want, dwant = run(z, tok, 1.0, 9, gl, gh)
    wide = torch.cat([z, z], 1)
    strided = (wide[:, :999], torch.cat([z[:, :1], z], 1)[:, 1:], z.t().contiguous().t())
    for v in strided:
        got, dz = run(v, tok, 1.0, 9, gl, gh)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(dz, dwant)
    # rows of more dimensions, and one alone
    y = z.view(2, 3, 999).clone().requires_grad_(True)
    got = LM.token_logprobs(y, tok.view(2, 3), top=9)
    assert got[0].shape == (2, 3) and got[3].shape == (2, 3, 9) and torch.equal(got[3].view(6, 9), want[3])
    (dz,) = torch.autograd.grad((got[0], got[1]), y, (gl.view(2, 3), gh.view(2, 3)))
    assert torch.equal(dz.view(6, 999), dwant)
    got = LM.token_logprobs(z[2], tok[2], top=9)
    assert got[0].shape == () and got[2].shape == (9,) and torch.equal(got[3], want[3][2])
    # the split of few rows does not change the alternatives, and every run has the same bits
    z, tok, gl, gh = inputs(1500, 20000, torch.bfloat16, dev, seed=8)
    many = LM.token_logprobs(z, tok, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = LM.token_logprobs(z, tok, top=20)
        few = LM.token_logprobs(z[:3], tok[:3], top=20)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(many, again):
        assert torch.equal(a, b)
    assert torch.equal(few[3], many[3][:3])


def test_offsets_beyond_32_bits(dev):
    from lifscan import hip_lm as LM
    z, tok, gl, gh = inputs(3, 5000, torch.bfloat16, dev, seed=9)
    far = torch.empty(2 ** 32 + 2 ** 20, dtype=torch.bfloat16, device=dev).as_strided((3, 5000), (2 ** 31, 1))
    far.copy_(z)
    a, da = run(far, tok, 1.0, 4, gl, gh)
    b, db = run(z, tok, 1.0, 4, gl, gh)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(da, db)


def test_rows_that_are_one_row(dev):
    """Expanded logits: read through a row stride of 0, and their gradient is summed."""
    from lifscan import hip_lm as LM
    z, tok, gl, gh = inputs(7, 700, torch.float32, dev, seed=14)
    y = z[:1].clone().requires_grad_(True)
    out = LM.token_logprobs(y.expand(7, 700), tok, top=3)
    (dz,) = torch.autograd.grad(out[:2], y, (gl, gh))
    want = reference(z[:1].expand(7, 700), tok, 1.0, 3, gl, gh)
    check(out, None, want, 700, 3)
    err = (dz.double().cpu() - want["dz"].sum(0)).abs()
    assert bool((err <= (64 + 700 / 64 + 7) * F * want["size"].sum(0) + 2.0 ** -126).all())


def test_calls_at_once_on_two_streams(dev):
    a, b = (inputs(5, 50000, torch.bfloat16, dev, seed=s) for s in (15, 16))
    want = [run(t[0], t[1], 1.0, 20, *t[2:]) for t in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for n in range(3):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = run(t[0], t[1], 1.0, 20, *t[2:])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g[0], w[0])) and torch.equal(g[1], w[1])


def test_empty(dev):
    from lifscan import hip_lm as LM
    z = torch.zeros(0, 7, device=dev, requires_grad=True)
    tok = torch.zeros(0, dtype=torch.int64, device=dev)
    out = LM.token_logprobs(z, tok, top=3)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 3), (0, 3)]
    assert torch.autograd.grad(out[0].sum() + out[1].sum(), z)[0].shape == (0, 7)


def test_graph_replays(dev):
    from lifscan import hip_lm as LM
    for rows, V in ((4, 20000), (1200, 300)):
        z, tok, gl, gh = inputs(rows, V, torch.bfloat16, dev, seed=10)
        zg = z.clone().requires_grad_(True)

        def work():
            out = LM.token_logprobs(zg, tok, temperature=0.9, top=5)
            return [o.detach() for o in out] + [*torch.autograd.grad(out[:2], zg, (gl, gh))]

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
                zg.normal_()
                tok.random_(0, V)
            graph.replay()
            torch.cuda.synchronize()
            kept = [o.clone() for o in outs]
            for a, b in zip(kept, work()):
                assert torch.equal(a, b)


def test_saved_tensors_that_come_back_changed(dev):
    from lifscan import hip_lm as LM
    z, tok, gl, gh = inputs(6, 500, torch.float32, dev, seed=11)
    _, want = run(z, tok, 1.0, 3, gl, gh)
    zg = z.clone().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0]):
        out = LM.token_logprobs(zg, tok, top=3)
    (dz,) = torch.autograd.grad(out[:2], zg, (gl, gh))
    assert torch.equal(dz, want)
    for change in (lambda t: t[:1], lambda t: t.half(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            out = LM.token_logprobs(zg, tok, top=3)
        with pytest.raises((ValueError, RuntimeError)):
            torch.autograd.grad(out[:2], zg, (gl, gh))


def test_refusals(dev):
    from lifscan import hip_lm as LM
    z, tok, *_ = inputs(4, 100, torch.float32, dev, seed=12)
    bad = [lambda: LM.token_logprobs(z.cpu(), tok.cpu()), lambda: LM.token_logprobs(z, tok.cpu()),
           lambda: LM.token_logprobs(z, tok[:3]), lambda: LM.token_logprobs(z, tok[:, None]), lambda: LM.token_logprobs(z, tok.float()),
           lambda: LM.token_logprobs(z.double(), tok), lambda: LM.token_logprobs(z, tok, temperature=0.0),
           lambda: LM.token_logprobs(z, tok, temperature=float("inf")), lambda: LM.token_logprobs(z, tok, temperature=float("nan")),
           lambda: LM.token_logprobs(z, tok, temperature=1e-39), lambda: LM.token_logprobs(z, tok, top=-1), lambda: LM.token_logprobs(z, tok, top=65),
           lambda: LM.token_logprobs(z[:, :20], tok, top=21), lambda: LM.token_logprobs(z[:, :0], tok),
           lambda: LM.token_logprobs(torch._neg_view(z), tok)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    y = z.clone().requires_grad_(True)
    out = LM.token_logprobs(y, tok, top=2)
    assert out[0].requires_grad and out[1].requires_grad and not out[2].requires_grad and not out[3].requires_grad
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out[0].sum(), y, create_graph=True)


def test_forward_mode_and_traces_are_refused(dev):
    import torch.autograd.forward_ad as fw
    from lifscan import hip_lm as LM
    z, tok, *_ = inputs(4, 100, torch.float32, dev, seed=13)
    call = lambda a: LM.token_logprobs(a, tok)[0]  # noqa: E731
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(fw.make_dual(z, z))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(call, (z,), check_trace=False)
    y = z.clone().requires_grad_(True)
    out = call(y)
    g = torch.randn_like(out)
    (want,) = torch.autograd.grad(out, y, -g, retain_graph=True)
    (got,) = torch.autograd.grad(out, y, torch._neg_view(g))
    assert torch.equal(got, want)
