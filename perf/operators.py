"""The operators of a spiking language model, as cases that can be timed and checked.

  step     linear attention with a decay for each head, one new token: the state updated in place
  prompt   linear attention over a prompt without gradients: outputs and the state after it
  attn     the same in a training step: outputs, final state, gradients of q, k, v and the first state
  norm     the norm after a block, its gate and residual scale, and the norm before the next block
  embed    embedding lookup with scaling, and the table's gradient
  distill  loss against a teacher's top logits, and the logits' gradient

own = False computes every operator in plain torch operations in 32 bits (one rounding at the end),
own = True through the framework's entry points.  Arrays are time-major, [T, B, ...], as in the rest
of the framework.  exact() follows the definitions token by token in 64 bits, gradients by the
adjoint formulas; the plain form works in chunks and takes its gradients from autograd.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
CHUNK = 64       # rows of a chunk in the plain linear attention
EPS = 1e-6       # of every norm
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _lm():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    at = os.path.join(root, "hard-resets-compose_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from lifscan import hip_linattn, hip_lm
    return hip_linattn, hip_lm


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # one sequence being generated, 8 heads of 64: launch and latency
        {"name": "step_one", "path": "step", "B": 1, "H": 8, "HK": 8, "DK": 64, "DV": 64, "dtype": "f32"},
        # a server's batch of 64 sequences, 16 heads of 128: the states stream through
        {"name": "step_batch", "path": "step", "B": 64, "H": 16, "HK": 16, "DK": 128, "DV": 128, "dtype": "bf16"},
        # a single long document read before generating: few heads, q/k/v views of one projection
        {"name": "prompt_long", "path": "prompt", "T": 32768, "B": 1, "H": 8, "HK": 8, "DK": 64, "DV": 128,
         "dtype": "bf16"},
        # the same operator in training, the largest: 4 sequences of 4096 tokens, 16 heads of 128
        {"name": "attn_wide", "path": "attn", "T": 4096, "B": 4, "H": 16, "HK": 16, "DK": 128, "DV": 128,
         "dtype": "bf16"},
        # ragged training in fp32 (the type of the neurons): odd length, shared keys and values, odd widths
        {"name": "attn_ragged", "path": "attn", "T": 1000, "B": 3, "H": 4, "HK": 2, "DK": 48, "DV": 80,
         "dtype": "f32"},
        # a training step's norms: 8192 tokens of 2048 channels
        {"name": "norm_train", "path": "norm", "rows": 8192, "D": 2048, "dtype": "bf16", "res": "bf16", "act": "silu",
         "train": True},
        # the norms of one decoding step: fp32 residual stream, bf16 block
        {"name": "norm_step", "path": "norm", "rows": 64, "D": 1024, "dtype": "bf16", "res": "f32", "act": "silu",
         "train": False},
        # token embedding of a training step: 16384 tokens of a Zipf vocabulary
        {"name": "embed_train", "path": "embed", "n": 16384, "V": 32000, "D": 1024, "dtype": "bf16"},
        # odd everything, fp32
        {"name": "embed_ragged", "path": "embed", "n": 1000, "V": 5003, "D": 257, "dtype": "f32"},
        # distillation of a training step: 64 teacher logits a token
        {"name": "distill_train", "path": "distill", "rows": 4096, "V": 32000, "K": 64, "tau": 2.0, "dtype": "bf16"},
        # few rows of a long odd vocabulary
        {"name": "distill_few", "path": "distill", "rows": 48, "V": 100003, "K": 16, "tau": 1.0, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm, odd ones as likely as even."""
    hi = max(lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    """A head's width: mostly the common ones, some that no tile divides."""
    return rng.choice([32, 64, 64, 128, 128, 256, rng.randrange(17, 160)])


def draw(rng):
    path = rng.choice(["step", "prompt", "attn", "attn", "norm", "embed", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if path in ("step", "prompt", "attn"):
        HK = rng.choice([1, 2, 4, 8, 16])
        H = HK * rng.choice([1, 1, 2, 4]) if HK < 16 else HK
        DK, DV = _width(rng), _width(rng)
        case = {"path": path, "H": H, "HK": HK, "DK": DK, "DV": DV, "dtype": dtype}
        if path == "step":
            return {**case, "B": _spread(rng, 1, max(1, min(128, 2 ** 24 // (H * DK * DV))))}
        most = 4096 * 4 * 16 * 128 * 128 // (4 if dtype == "f32" else 1)  # fp32 works through four times the cost
        B = _spread(rng, 1, 8)
        T = _spread(rng, 1, max(1, min(32768 if path == "prompt" else 4096, most // (H * DK * DV * B))))
        return {**case, "T": T, "B": B}
    if path == "norm":
        D = _spread(rng, 64, 8192)
        return {"path": path, "rows": _spread(rng, 1, min(16384, 2 ** 24 // D)), "D": D, "dtype": dtype,
                "res": rng.choice(["f32", dtype]), "act": rng.choice(["silu", "sigmoid"]),
                "train": rng.choice([True, True, False])}
    if path == "embed":
        D = _spread(rng, 16, 4096)
        return {"path": path, "n": _spread(rng, 1, min(65536, 2 ** 24 // D)), "V": _spread(rng, 100, min(100000, 2 ** 25 // D)),
                "D": D, "dtype": dtype}
    V = _spread(rng, 100, 130000)
    return {"path": path, "rows": _spread(rng, 1, min(8192, 2 ** 26 // V)), "V": V,
            "K": rng.choice([1, 5, 16, 64, 100]), "tau": rng.choice([1.0, 2.0, 3.5]), "dtype": dtype}


def work(case):
    c, e = case, SIZES[case["dtype"]]
    if c["path"] in ("step", "prompt", "attn"):
        tokens = c["B"] * c.get("T", 1)
        qo, kv = c["H"] * (c["DK"] + c["DV"]), c["HK"] * (c["DK"] + c["DV"])
        state = c["B"] * c["H"] * c["DK"] * c["DV"]
        if c["path"] == "step":
            return {"bytes": 8 * state + e * tokens * (qo + kv), "flops": 5 * state}
        flops = 5.0 * tokens * c["H"] * c["DK"] * c["DV"]  # update and read of the state, token by token
        if c["path"] == "prompt":
            return {"bytes": e * tokens * (qo + kv) + 8 * state, "flops": flops}
        # forward as above; backward reads q, k, v, do and dS_T, writes dq, dk, dv and ds0
        return {"bytes": e * tokens * ((qo + kv) + (qo + kv) + c["H"] * c["DK"] + kv) + 20 * state, "flops": 3.2 * flops}
    if c["path"] == "norm":
        n, r = c["rows"] * c["D"], SIZES[c["res"]]
        fwd = n * (2 * r + 3 * e)                  # x, y, gate read, x_new, z written
        if not c["train"]:
            return {"bytes": fwd + 3 * 4 * c["D"], "flops": 15 * n}
        return {"bytes": fwd + n * (3 * r + 5 * e) + 6 * 4 * c["D"], "flops": 55 * n}
    if c["path"] == "embed":
        n, D = c["n"], c["D"]
        rows = min(n, c["V"])                      # at most: how many differ depends on the tokens
        return {"bytes": 2 * 8 * n + e * D * (rows + 2 * n + c["V"]), "flops": 3 * n * D}
    return {"bytes": 3 * c["rows"] * c["V"] * e + c["rows"] * c["K"] * 24, "flops": 12 * c["rows"] * c["V"]}


# ----------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["path"] in ("step", "prompt", "attn"):
        B, H, HK, DK, DV = (c[k] for k in ("B", "H", "HK", "DK", "DV"))
        T = c.get("T", 1)
        # decays from 7/8 to 1 - 2^-10, another one for each head
        s["beta"] = 1 - torch.exp2(-torch.linspace(3, 10, H, device=DEVICE)) * (0.9 + 0.1 * torch.rand(H, generator=g, device=DEVICE))
        s["scale"] = DK ** -0.5
        # q, k and v leave one projection and are views of its output
        x = _normal(g, T, B, H * DK + HK * (DK + DV)).to(dt)
        q, k, v = x.split([H * DK, HK * DK, HK * DV], -1)
        s["q"], s["k"], s["v"] = q.unflatten(-1, (H, DK)), k.unflatten(-1, (HK, DK)), v.unflatten(-1, (HK, DV))
        s["s0"] = 4 * _normal(g, B, H, DK, DV)
        if c["path"] == "step":
            for k in ("q", "k", "v"):
                s[k] = s[k][0]
        if c["path"] == "attn":
            s["do"] = _normal(g, T, B, H, DV).to(dt)
            s["ds"] = 0.1 * _normal(g, B, H, DK, DV)
            for k in ("q", "k", "v", "s0"):
                s[k].requires_grad_(True)
    elif c["path"] == "norm":
        n, D, res = c["rows"], c["D"], DTYPES[c["res"]]
        s["x"] = (2 * _normal(g, n, D)).to(res)
        s["y"] = (0.5 * _normal(g, n, D)).to(dt)
        s["gate"] = _normal(g, n, D).to(dt)
        s["w_post"], s["w_pre"] = 1 + 0.1 * _normal(g, D), 1 + 0.1 * _normal(g, D)
        s["res_scale"] = 0.3 + 0.05 * _normal(g, D)
        if c["train"]:
            s["gx"], s["gz"] = _normal(g, n, D).to(res), _normal(g, n, D).to(dt)
            for k in ("x", "y", "gate", "w_post", "w_pre", "res_scale"):
                s[k].requires_grad_(True)
    elif c["path"] == "embed":
        n, V, D = c["n"], c["V"], c["D"]
        # Zipf: the most frequent token is some seven in a hundred of a 32000-word text
        u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
        s["tokens"] = (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)
        s["weight"] = _normal(g, V, D).to(dt).requires_grad_(True)
        s["scale"] = math.sqrt(D)
        s["padding"] = min(3, V - 1)
        s["dout"] = (0.02 * _normal(g, n, D)).to(dt)
    else:
        n, V, K = c["rows"], c["V"], c["K"]
        z = 2.5 * _normal(g, n, V)
        s["logits"] = z.to(dt)
        # a teacher that mostly agrees: its top logits are those of a noisier copy
        top = (z + _normal(g, n, V)).topk(min(K, V), -1)
        s["values"], s["index"] = top.values.to(dt), top.indices
        # tokens that the teacher was not asked about, and lists that end early
        cut = torch.randint(0, 2 * s["index"].shape[1] + 1, (n, 1), generator=g, device=DEVICE)
        s["index"].masked_fill_(torch.arange(s["index"].shape[1], device=DEVICE) >= cut, -1)
        s["weight"] = torch.rand(n, generator=g, device=DEVICE) / n
        s["logits"].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------- plain forms
def _heads(x, H):
    """[T, B, Hx, D] of any type -> fp32 [B, H, T, D], shared heads repeated."""
    x = x.float()
    return x.repeat_interleave(H // x.shape[2], 2).permute(1, 2, 0, 3)


def _plain_attention(q, k, v, beta, s0, scale):
    """Products inside chunks, and one product that carries the chunks' sums to later chunks."""
    T, B = q.shape[:2]
    H = beta.numel()
    DK, DV = q.shape[-1], v.shape[-1]
    lb = beta.log()
    q, k, v = _heads(q, H), _heads(k, H), _heads(v, H)
    left = torch.arange(T - 1, -1, -1, device=q.device)
    s_end = (k * (lb[:, None] * left).exp()[..., None]).transpose(-1, -2) @ v + s0 * (lb * T).exp()[:, None, None]
    C = min(CHUNK, T)
    n = -(-T // C)
    pad = (0, 0, 0, n * C - T)
    q, k, v = (torch.nn.functional.pad(t, pad).reshape(B, H, n, C, -1) for t in (q, k, v))
    i = torch.arange(C, device=q.device)
    far = i[:, None] - i
    mask = torch.where(far >= 0, (lb[:, None, None] * far).exp(), 0.0)[:, None]
    inside = ((q @ k.transpose(-1, -2)) * mask) @ v
    sums = (k * (lb[:, None] * (C - 1 - i)).exp()[:, None, :, None]).transpose(-1, -2) @ v
    m = torch.arange(n, device=q.device)
    gap = m[:, None] - 1 - m
    carry = torch.where(gap >= 0, (lb[:, None, None] * (C * gap)).exp(), 0.0)
    first = (lb[:, None] * (C * m)).exp()[..., None, None] * s0[:, :, None]
    starts = (carry @ sums.reshape(B, H, n, DK * DV)).reshape(B, H, n, DK, DV) + first
    before = (q * (lb[:, None] * (i + 1)).exp()[:, None, :, None]) @ starts
    o = scale * (inside + before).reshape(B, H, n * C, DV)[:, :, :T]
    return o.permute(2, 0, 1, 3), s_end


def _plain_norm(x):
    return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()


def _plain_block_norm(x, y, gate, w_post, w_pre, res_scale, act):
    x, y, gate = x.float(), y.float(), gate.float()
    a = gate * gate.sigmoid() if act == "silu" else gate.sigmoid()
    x_new = x + res_scale * (a * (_plain_norm(y) * w_post))
    return x_new, _plain_norm(x_new) * w_pre


def _plain_embed(tokens, weight, scale, padding):
    rows = weight.float()[tokens] * scale
    return rows.masked_fill((tokens == padding)[:, None], 0.0)


def _plain_distill(logits, values, index, tau):
    there = index >= 0
    t = torch.where(there, values.float() / tau, -math.inf)
    some = there.any(-1, keepdim=True)
    p = torch.where(some, t, 0.0).softmax(-1) * there
    z = logits.float() / tau
    logq = z.gather(-1, index.clamp(min=0)) - z.logsumexp(-1, keepdim=True)
    return tau * tau * torch.where(p > 0, p * (p.clamp(min=1e-38).log() - logq), 0.0).sum(-1)


def _grads(outs, ins, gouts):
    return torch.autograd.grad(outs, ins, gouts)


def _run_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["path"] == "step":
        H = s["beta"].numel()
        q, k, v = (t.float().repeat_interleave(H // t.shape[1], 1) for t in (s["q"], s["k"], s["v"]))
        s["s0"].mul_(s["beta"][:, None, None]).add_(k[..., :, None] * v[..., None, :])
        return (s["scale"] * (q[..., None, :] @ s["s0"])[..., 0, :]).to(dt), s["s0"]
    if c["path"] == "prompt":
        o, s_end = _plain_attention(s["q"], s["k"], s["v"], s["beta"], s["s0"], s["scale"])
        return o.to(dt), s_end
    if c["path"] == "attn":
        ins = [s[k] for k in ("q", "k", "v", "s0")]
        o, s_end = _plain_attention(*ins[:3], s["beta"], ins[3], s["scale"])
        return (o.detach().to(dt), s_end.detach(), *_grads((o, s_end), ins, (s["do"].float(), s["ds"])))
    if c["path"] == "norm":
        names = ("x", "y", "gate", "w_post", "w_pre", "res_scale")
        ins = [s[k] for k in names]
        x_new, z = _plain_block_norm(*ins, c["act"])
        outs = [x_new.detach().to(DTYPES[c["res"]]), z.detach().to(dt)]
        if c["train"]:
            outs += _grads((x_new, z), ins, (s["gx"].float(), s["gz"].float()))
        return outs
    if c["path"] == "embed":
        out = _plain_embed(s["tokens"], s["weight"], s["scale"], s["padding"])
        return [out.detach().to(dt), *_grads(out, s["weight"], s["dout"].float())]
    loss = _plain_distill(s["logits"], s["values"], s["index"], c["tau"])
    return [loss.detach(), *_grads(loss, s["logits"], s["weight"])]


def _run_own(s):
    LA, LM = _lm()
    c = s["case"]
    if c["path"] == "step":
        return LA.lin_attn_step(s["q"], s["k"], s["v"], s["beta"], s["s0"], scale=s["scale"]), s["s0"]
    if c["path"] == "prompt":
        return LA.lin_attn(s["q"], s["k"], s["v"], s["beta"], s0=s["s0"], scale=s["scale"])
    if c["path"] == "attn":
        ins = [s[k] for k in ("q", "k", "v", "s0")]
        o, s_end = LA.lin_attn(*ins[:3], s["beta"], s0=ins[3], scale=s["scale"])
        return (o.detach(), s_end.detach(), *_grads((o, s_end), ins, (s["do"], s["ds"])))
    if c["path"] == "norm":
        x, y, gate, w_post, w_pre, res_scale = ins = [s[k] for k in ("x", "y", "gate", "w_post", "w_pre", "res_scale")]
        x_new, z = LM.block_norm(x, y, w_post, w_pre, gate=gate, res_scale=res_scale, eps=EPS, act=c["act"])
        outs = [x_new.detach(), z.detach()]
        if c["train"]:
            outs += _grads((x_new, z), ins, (s["gx"], s["gz"]))
        return outs
    if c["path"] == "embed":
        out = LM.embed(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
        return [out.detach(), *_grads(out, s["weight"], s["dout"])]
    loss = LM.distill_topk(s["logits"], s["values"], s["index"], temperature=c["tau"])
    return [loss.detach(), *_grads(loss, s["logits"], s["weight"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------- 64 bits
def _exact_attention(s, c):
    H = s["beta"].numel()
    step = c["path"] == "step"
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    if step:
        q, k, v = q[None], k[None], v[None]
    per = [H // t.shape[2] for t in (q, k, v)]
    q, k, v = (t.repeat_interleave(r, 2) for t, r in zip((q, k, v), per))
    beta, scale = s["beta"].double()[:, None, None], s["scale"]
    S = s["s0"].detach().double().clone()
    train = c["path"] == "attn"
    do = s["do"].double() if train else None
    o = torch.empty_like(v)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v)) if train else (None, None, None)
    for t in range(q.shape[0]):
        S = beta * S + k[t][..., :, None] * v[t][..., None, :]
        o[t] = scale * (S * q[t][..., :, None]).sum(-2)
        if train:
            dq[t] = scale * (S * do[t][..., None, :]).sum(-1)
    if step:
        return o[0], S
    if not train:
        return o, S
    E = s["ds"].double().clone()
    for t in range(q.shape[0] - 1, -1, -1):
        G = E + scale * q[t][..., :, None] * do[t][..., None, :]
        dk[t] = (G * v[t][..., None, :]).sum(-1)
        dv[t] = (G * k[t][..., :, None]).sum(-2)
        E = beta * G
    dq, dk, dv = (d.unflatten(2, (-1, r)).sum(3) for d, r in zip((dq, dk, dv), per))
    return o, S, dq, dk, dv, E


def _exact_norm(s, c):
    x, y, gate, w_post, w_pre, a = (s[k].detach().double() for k in ("x", "y", "gate", "w_post", "w_pre", "res_scale"))
    D = x.shape[1]
    sg = 1 / (1 + torch.exp(-gate))
    act, dact = (gate * sg, sg * (1 + gate * (1 - sg))) if c["act"] == "silu" else (sg, sg * (1 - sg))
    ry = 1 / torch.sqrt((y * y).sum(1, keepdim=True) / D + EPS)
    n = y * ry * w_post
    h = act * n
    xn = x + a * h
    rx = 1 / torch.sqrt((xn * xn).sum(1, keepdim=True) / D + EPS)
    z = xn * rx * w_pre
    if not c["train"]:
        return [xn, z]
    gx, gz = s["gx"].double(), s["gz"].double()
    u = gz * w_pre
    dx = gx + rx * (u - xn * rx * rx * (u * xn).sum(1, keepdim=True) / D)
    dh = dx * a
    dn = dh * act
    m = dn * w_post
    dy = ry * (m - y * ry * ry * (m * y).sum(1, keepdim=True) / D)
    return [xn, z, dx, dy, dh * n * dact, (dn * y * ry).sum(0), (gz * xn * rx).sum(0), (dx * h).sum(0)]


def _exact_embed(s, c):
    tok, w, keep = s["tokens"], s["weight"].detach().double(), (s["tokens"] != s["padding"]).double()[:, None]
    out = torch.index_select(w, 0, tok) * (s["scale"] * keep)
    dw = torch.zeros_like(w)
    order = torch.argsort(tok, stable=True)
    sums = torch.cat([dw.new_zeros(1, w.shape[1]), (s["dout"].double() * keep * s["scale"])[order].cumsum(0)])
    end = torch.bincount(tok, minlength=w.shape[0]).cumsum(0)
    begin = torch.cat([end.new_zeros(1), end[:-1]])
    return [out, sums[end] - sums[begin]]


def _exact_distill(s, c):
    z, tau = s["logits"].detach().double() / c["tau"], c["tau"]
    there = (s["index"] >= 0).double()
    e = torch.exp((s["values"].double() - s["values"].double().max(1, keepdim=True).values) / tau) * there
    mass = e.sum(1, keepdim=True)
    p = torch.where(mass > 0, e / mass.clamp(min=1e-300), 0.0)
    top = z.max(1, keepdim=True).values
    w = torch.exp(z - top)
    total = w.sum(1, keepdim=True)
    at = s["index"].clamp(min=0)
    logq = torch.gather(z, 1, at) - top - torch.log(total)
    loss = tau * tau * (torch.special.xlogy(p, p) - p * logq).sum(1)
    dz = w / total * p.sum(1, keepdim=True)
    dz.scatter_add_(1, at, -p)
    return [loss, dz * (s["weight"].double()[:, None] * tau)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] in ("step", "prompt", "attn"):
        return _exact_attention(s, case)
    with torch.no_grad():
        return {"norm": _exact_norm, "embed": _exact_embed, "distill": _exact_distill}[case["path"]](s, case)
