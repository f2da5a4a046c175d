"""More operators of a spiking language model, as cases that can be timed and checked.

  scan    a gated linear recurrence over a sequence: a decay for each channel and token
  step    the same for one new token: the state updated in place
  rotate  norms of queries and keys for each head, and their rotation by position, in one pass
  score   log probabilities of given tokens, the entropy and the most likely alternatives

own = False computes every operator in plain torch operations in 32 bits (angles in 64; one rounding at
the end), own = True through the framework's entry points.  Arrays are time-major, [T, B, ...].  exact()
follows the definitions in 64 bits, the recurrence token by token, gradients by the adjoint formulas; the
plain form scans by doubling and takes its gradients from autograd.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
BASE = 10000.0   # of the rotation's frequencies
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _lm():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    at = os.path.join(root, "hard-resets-compose_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from lifscan import hip_gated, hip_linattn, hip_lm
    return hip_gated, hip_linattn, hip_lm


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # training: 4 sequences of 4096 tokens, 2048 channels
        {"name": "scan_train", "path": "scan", "T": 4096, "B": 4, "D": 2048, "dtype": "bf16", "decay": "sigmoid",
         "mix": True, "starts": False, "train": True},
        # a single long document read before generating
        {"name": "scan_long", "path": "scan", "T": 32768, "B": 1, "D": 1024, "dtype": "bf16", "decay": "log",
         "mix": True, "starts": False, "train": False},
        # training on packed documents of odd sizes in fp32, the type of the neurons
        {"name": "scan_packed", "path": "scan", "T": 1000, "B": 3, "D": 257, "dtype": "f32", "decay": "sigmoid",
         "mix": False, "starts": True, "train": True},
        # one sequence being generated: launch and latency
        {"name": "step_one", "path": "step", "B": 1, "D": 512, "dtype": "f32", "decay": "sigmoid", "mix": True},
        # a server's batch of 256 sequences
        {"name": "step_batch", "path": "step", "B": 256, "D": 4096, "dtype": "bf16", "decay": "sigmoid", "mix": True},
        # training: queries and keys of 8192 tokens, 16 heads of 128 and 4 shared ones
        {"name": "rotate_train", "path": "rotate", "T": 4096, "B": 2, "H": 16, "HK": 4, "D": 128, "rot": 128,
         "pairs": "halves", "norm": True, "far": False, "dtype": "bf16", "train": True},
        # one token each of 64 sequences, far into them
        {"name": "rotate_step", "path": "rotate", "T": 1, "B": 64, "H": 16, "HK": 16, "D": 64, "rot": 64,
         "pairs": "halves", "norm": True, "far": True, "dtype": "f16", "train": False},
        # odd everything, fp32: half of each head rotated, as neighbouring pairs
        {"name": "rotate_ragged", "path": "rotate", "T": 1003, "B": 3, "H": 6, "HK": 2, "D": 80, "rot": 36,
         "pairs": "neighbours", "norm": True, "far": False, "dtype": "f32", "train": True},
        # training on given tokens: loss and gradient of 4096 tokens
        {"name": "score_train", "path": "score", "rows": 4096, "V": 32000, "K": 0, "tau": 1.0, "banned": 0.0,
         "dtype": "bf16", "train": True},
        # a text scored, with five alternatives at each token
        {"name": "score_text", "path": "score", "rows": 2048, "V": 32000, "K": 5, "tau": 1.0, "banned": 0.0,
         "dtype": "bf16", "train": False},
        # what a server answers with: 24 sequences, a long odd vocabulary of which a part is not allowed
        {"name": "score_serve", "path": "score", "rows": 24, "V": 100003, "K": 20, "tau": 0.7, "banned": 0.3,
         "dtype": "f32", "train": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm, odd ones as likely as even."""
    hi = max(lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(["scan", "scan", "step", "rotate", "rotate", "score", "score"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    most = 2 ** 25 if dtype != "f32" else 2 ** 24  # elements, so that fp32 moves no more bytes
    if path in ("scan", "step"):
        D, B = _spread(rng, 16, 4096), _spread(rng, 1, 16 if path == "scan" else 512)
        if rng.random() < 0.6:
            D = -(-D // 64) * 64
        case = {"path": path, "B": B, "D": D, "dtype": dtype, "decay": rng.choice(["sigmoid", "log"]),
                "mix": rng.choice([True, False])}
        if path == "step":
            return case
        return {**case, "T": _spread(rng, 1, max(1, min(65536, most // (B * D)))), "starts": rng.choice([True, False]),
                "train": rng.choice([True, True, False])}
    if path == "rotate":
        HK = rng.choice([1, 2, 4, 8, 16])
        H = HK * rng.choice([1, 2, 4])
        D = rng.choice([32, 64, 64, 128, 128, 256, 2 * rng.randrange(8, 100)])
        rot = rng.choice([D, D, 2 * rng.randrange(1, D // 2 + 1)])
        B = _spread(rng, 1, 64)
        return {"path": path, "T": _spread(rng, 1, max(1, min(32768, most // (B * (H + HK) * D)))), "B": B, "H": H, "HK": HK,
                "D": D, "rot": rot, "pairs": rng.choice(["halves", "halves", "neighbours"]),
                "norm": rng.choice([True, True, False]), "far": rng.choice([True, False]), "dtype": dtype,
                "train": rng.choice([True, True, False])}
    V = _spread(rng, 100, 130000)
    return {"path": path, "rows": _spread(rng, 1, min(8192, 2 * most // V)), "V": V, "K": rng.choice([0, 1, 5, 20]),
            "tau": rng.choice([1.0, 0.7, 2.0]), "banned": rng.choice([0.0, 0.0, 0.3]), "dtype": dtype,
            "train": rng.choice([True, False])}


def work(case):
    c, e = case, SIZES[case["dtype"]]
    if c["path"] == "step":
        n = c["B"] * c["D"]
        return {"bytes": (3 * e + 8) * n, "flops": 10 * n}
    if c["path"] == "scan":
        n, rows = c["T"] * c["B"] * c["D"], c["T"] * c["B"]
        state = 4 * c["B"] * c["D"]
        mask = rows if c["starts"] else 0
        if not c["train"]:
            return {"bytes": 3 * e * n + 2 * state + mask, "flops": 10 * n}
        # forward as above; backward reads x, gate, dh and dh_end, writes dx, dgate and dh0
        return {"bytes": 8 * e * n + 4 * state + 2 * mask, "flops": 30 * n}
    if c["path"] == "rotate":
        rows = c["T"] * c["B"]
        n = rows * (c["H"] + c["HK"]) * c["D"]
        small = 8 * rows + 4 * c["rot"] + (8 * c["D"] if c["norm"] else 0)
        if not c["train"]:
            return {"bytes": 2 * e * n + small, "flops": 8 * n}
        # without norms the gradients are rotations of the outputs' gradients
        return {"bytes": (5 if c["norm"] else 4) * e * n + 2 * small, "flops": 24 * n}
    n = c["rows"] * c["V"]
    small = c["rows"] * (16 + 12 * c["K"])
    return {"bytes": (3 if c["train"] else 1) * e * n + small, "flops": (12 if c["train"] else 6) * n}


# ----------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device=DEVICE, dtype=torch.float32)


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["path"] in ("scan", "step"):
        T, B, D = c.get("T", 1), c["B"], c["D"]
        # values and gates leave one projection and are views of its output; decays from about 0.6 to 0.998
        both = _normal(g, T, B, 2 * D)
        both[..., D:] += torch.linspace(0.5, 6.0, D, device=DEVICE)
        if c["decay"] == "log":
            both[..., D:] = -torch.exp(-both[..., D:])
        x, gate = both.to(dt).split([D, D], -1)
        s["x"], s["gate"] = x, gate
        s["h0"] = _normal(g, B, D)
        if c["path"] == "step":
            s["x"], s["gate"] = x[0], gate[0]
            return s
        # documents of some 200 tokens packed one behind the other
        s["starts"] = (_uniform(g, T, B) < 0.005) if c["starts"] else None
        if c["train"]:
            s["dh"], s["dend"] = _normal(g, T, B, D).to(dt), _normal(g, B, D)
            for k in ("x", "gate", "h0"):
                s[k].requires_grad_(True)
    elif c["path"] == "rotate":
        T, B, H, HK, D = (c[k] for k in ("T", "B", "H", "HK", "D"))
        q, k = _normal(g, T, B, (H + HK) * D).to(dt).split([H * D, HK * D], -1)
        s["q"], s["k"] = q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D))
        s["inv_freq"] = BASE ** -(torch.arange(c["rot"] // 2, device=DEVICE, dtype=torch.float64) * 2 / c["rot"])
        # sequences that began elsewhere, or all from their first token
        far = torch.randint(0, 2 ** 20, (B,), generator=g, device=DEVICE)
        at = torch.arange(T, device=DEVICE)
        s["positions"] = at[:, None] + far if c["far"] else at
        s["w_q"] = 1 + 0.1 * _normal(g, D) if c["norm"] else None
        s["w_k"] = 1 + 0.1 * _normal(g, D) if c["norm"] else None
        if c["train"]:
            s["dq"], s["dk"] = _normal(g, T, B, H, D).to(dt), _normal(g, T, B, HK, D).to(dt)
            for k in ("q", "k", "w_q", "w_k"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    else:
        n, V = c["rows"], c["V"]
        z = 2.5 * _normal(g, n, V)
        if c["banned"]:
            z.masked_fill_(_uniform(g, n, V) < c["banned"], -math.inf)
        s["logits"] = z.to(dt)
        # the tokens that followed: drawn from a sharper distribution; one in twenty is padding
        s["tokens"] = (1.5 * z).sub_(_uniform(g, n, V).clamp_(min=1e-30).log_().neg_().log_()).argmax(-1)
        s["tokens"].masked_fill_(_uniform(g, n) < 0.05, -1)
        if c["train"]:
            s["g_logp"], s["g_entropy"] = -_uniform(g, n) / n, 0.01 * _uniform(g, n) / n
            s["logits"].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_decay(gate, decay):
    """(a, 1 - a)"""
    if decay == "sigmoid":
        return gate.sigmoid(), (-gate).sigmoid()
    gate = gate.clamp(max=0.0)
    return gate.exp(), -gate.expm1()


def _plain_scan(x, gate, h0, starts, decay, mix):
    """Spans that double in each round: after it every row holds the sum over the last 2, 4, 8, ... rows."""
    T = x.shape[0]
    a, rest = _plain_decay(gate.float(), decay)
    h = rest * x.float() if mix else x.float()
    if starts is not None:
        a = a.masked_fill(starts[..., None], 0.0)
    h = torch.cat([h[:1] + a[:1] * h0, h[1:]])
    span = 1
    while span < T:
        h = torch.cat([h[:span], h[span:] + a[span:] * h[:-span]])
        if 2 * span < T:
            a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return h, h[-1]


def _plain_rotate(x, weight, cos, sin, rot, pairs):
    x = x.float()
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
    y, rest = x[..., :rot], x[..., rot:]
    if pairs == "halves":
        u, v = y[..., :rot // 2], y[..., rot // 2:]
        return torch.cat([u * cos - v * sin, u * sin + v * cos, rest], -1)
    u, v = y[..., ::2], y[..., 1::2]
    return torch.cat([torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2), rest], -1)


def _angles(s):
    """cos and sin as [T, 1 or B, 1, rot / 2]."""
    p = s["positions"]
    angle = (p if p.dim() == 2 else p[:, None]).double()[..., None, None] * s["inv_freq"]
    return angle.cos().float(), angle.sin().float()


def _plain_score(logits, tokens, tau, K):
    z = logits.float() / tau
    with torch.no_grad():
        m = z.max(-1, keepdim=True).values
    z = z - m
    l = z.exp().sum(-1, keepdim=True).log()
    there = tokens >= 0
    logp = (z.gather(-1, tokens.clamp(min=0)[:, None]) - l)[:, 0].masked_fill(~there, 0.0)
    p = (z - l).exp()
    entropy = l[:, 0] - (p * torch.where(p > 0, z, 0.0)).sum(-1)
    if K == 0:
        return logp, entropy
    with torch.no_grad():
        # the order of the values as whole numbers, and below it the ids from the last: no two are alike
        bits = (logits.float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
        V = z.shape[1]
        index = V - 1 - torch.topk(order * 2 ** 24 + torch.arange(V - 1, -1, -1, device=z.device), K, -1).values % 2 ** 24
        top = z.gather(-1, index) - l
    return logp, entropy, top, index


def _grads(outs, ins, gouts):
    return torch.autograd.grad(outs, ins, gouts)


def _run_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["path"] == "step":
        a, rest = _plain_decay(s["gate"].float(), c["decay"])
        s["h0"].mul_(a).add_(rest * s["x"].float() if c["mix"] else s["x"].float())
        return s["h0"].to(dt), s["h0"]
    if c["path"] == "scan":
        ins = [s[k] for k in ("x", "gate", "h0")]
        h, end = _plain_scan(*ins, s["starts"], c["decay"], c["mix"])
        out = [h.detach().to(dt), end.detach()]
        if c["train"]:
            out += _grads((h, end), ins, (s["dh"].float(), s["dend"]))
        return out
    if c["path"] == "rotate":
        cos, sin = _angles(s)
        q = _plain_rotate(s["q"], s["w_q"], cos, sin, c["rot"], c["pairs"])
        k = _plain_rotate(s["k"], s["w_k"], cos, sin, c["rot"], c["pairs"])
        out = [q.detach().to(dt), k.detach().to(dt)]
        if c["train"]:
            ins = [s[n] for n in ("q", "k", "w_q", "w_k") if s[n] is not None]
            out += _grads((q, k), ins, (s["dq"].float(), s["dk"].float()))
        return out
    out = _plain_score(s["logits"], s["tokens"], c["tau"], c["K"])
    if c["train"]:
        grad = _grads(out[:2], s["logits"], (s["g_logp"], s["g_entropy"]))
        return [o.detach() for o in out] + [*grad]
    return [*out]


def _run_own(s):
    G, LA, LM = _lm()
    c = s["case"]
    if c["path"] == "step":
        return G.gated_scan_step(s["x"], s["gate"], s["h0"], decay=c["decay"], mix=c["mix"]), s["h0"]
    if c["path"] == "scan":
        ins = [s[k] for k in ("x", "gate", "h0")]
        h, end = G.gated_scan(*ins, starts=s["starts"], decay=c["decay"], mix=c["mix"])
        out = [h.detach(), end.detach()]
        if c["train"]:
            out += _grads((h, end), ins, (s["dh"], s["dend"]))
        return out
    if c["path"] == "rotate":
        q, k = LA.norm_rotate(s["q"], s["k"], s["positions"], s["inv_freq"], s["w_q"], s["w_k"], eps=EPS,
                              pairs=c["pairs"])
        out = [q.detach(), k.detach()]
        if c["train"]:
            ins = [s[n] for n in ("q", "k", "w_q", "w_k") if s[n] is not None]
            out += _grads((q, k), ins, (s["dq"], s["dk"]))
        return out
    out = LM.token_logprobs(s["logits"], s["tokens"], temperature=c["tau"], top=c["K"])
    if c["train"]:
        grad = _grads(out[:2], s["logits"], (s["g_logp"], s["g_entropy"]))
        return [o.detach() for o in out] + [*grad]
    return [*out]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------- 64 bits
def _exact_decay(gate, decay):
    """(a, 1 - a, da/dgate)"""
    if decay == "sigmoid":
        a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
        return a, rest, a * rest
    a = torch.exp(torch.minimum(gate, torch.zeros_like(gate)))
    return a, 1 - a, torch.where(gate > 0, 0.0, a)


def _exact_scan(s, c):
    x, gate, h = (s[k].detach().double() for k in ("x", "gate", "h0"))
    if c["path"] == "step":
        a, rest, _ = _exact_decay(gate, c["decay"])
        h = a * h + (rest * x if c["mix"] else x)
        return h, h
    T = x.shape[0]
    a, rest, slope = _exact_decay(gate, c["decay"])
    keep = torch.ones_like(a[..., :1]) if s["starts"] is None else 1 - s["starts"].double()[..., None]
    a = a * keep
    weight = rest if c["mix"] else torch.ones_like(rest)
    out, before = torch.empty_like(x), torch.empty_like(x)
    for t in range(T):
        before[t] = h * keep[t]
        h = a[t] * h + weight[t] * x[t]
        out[t] = h
    if not c["train"]:
        return [out, h]
    dh, E = s["dh"].double(), s["dend"].double().clone()
    adjoint = torch.empty_like(x)
    for t in range(T - 1, -1, -1):
        E = E + dh[t]
        adjoint[t] = E
        E = a[t] * E
    return [out, h, weight * adjoint, adjoint * (before - x if c["mix"] else before) * slope, E]


def _exact_rotate(s, c):
    T, B, rot, D = c["T"], c["B"], c["rot"], c["D"]
    p = s["positions"].double()
    p = p if p.dim() == 2 else p[:, None].expand(T, B)
    angle = p[..., None, None] * s["inv_freq"]
    i = torch.arange(rot // 2, device=p.device)
    first, second = (i, i + rot // 2) if c["pairs"] == "halves" else (2 * i, 2 * i + 1)

    def turn(y, angle):
        z = y.clone()
        z[..., first] = y[..., first] * torch.cos(angle) - y[..., second] * torch.sin(angle)
        z[..., second] = y[..., second] * torch.cos(angle) + y[..., first] * torch.sin(angle)
        return z

    outs, grads, sums = [], [], []
    for name in "qk":
        x, w = s[name].detach().double(), s["w_" + name]
        if w is None:
            r, w1 = torch.ones_like(x[..., :1]), torch.ones(D, device=p.device, dtype=torch.float64)
        else:
            w1 = w.detach().double()
            r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
        outs.append(turn(x * r * w1, angle))
        if c["train"]:
            u = turn(s["d" + name].double(), -angle)
            if w is None:
                grads.append(u)
            else:
                m = u * w1
                grads.append(r * (m - x * r * r * (m * x).sum(-1, keepdim=True) / D))
                sums.append((u * x * r).sum((0, 1, 2)))
    return outs + grads + sums


def _exact_score(s, c):
    z = s["logits"].detach().double() / c["tau"]
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    logp_all = z - top - torch.log(total)
    entropy = -torch.special.xlogy(p, p).sum(1)
    y = s["tokens"]
    there = (y >= 0).double()
    at = y.clamp(min=0)[:, None]
    logp = torch.gather(logp_all, 1, at)[:, 0]
    out = [torch.where(y >= 0, logp, 0.0), entropy]
    if c["K"]:
        # selected one after the other, each time the first of the largest
        left, picked = s["logits"].detach().double().clone(), []
        ids = torch.arange(z.shape[1], device=z.device)
        for _ in range(c["K"]):
            best = left.max(1, keepdim=True).values
            first = torch.where(left == best, ids, z.shape[1]).min(1, keepdim=True).values
            picked.append(first)
            left.scatter_(1, first, float("nan"))
            left = torch.where(torch.isnan(left), -math.inf, left)
        index = torch.cat(picked, 1)
        out += [torch.gather(logp_all, 1, index), index]
    if c["train"]:
        gl, gh = s["g_logp"].double() * there, s["g_entropy"].double()
        d = -p * gl[:, None] - gh[:, None] * (torch.special.xlogy(p, p) + p * entropy[:, None])
        d.scatter_add_(1, at, gl[:, None])
        out.append(d / c["tau"])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"scan": _exact_scan, "step": _exact_scan, "rotate": _exact_rotate, "score": _exact_score}[case["path"]](s, case)
