"""GPU: the spiking language model with a gated recurrence or with normed and rotated heads, its scores and its
likelihood loss: the operators run together, in training, whole, in pieces and token by token."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FORMS = [dict(mixer="gated"), dict(rotary=True), dict()]
IDS = ["gated", "rotary", "attention"]


def model(dev, seed=0, dtype=torch.float32, **kw):
    from lifscan.spikelm import SpikeLM
    torch.manual_seed(seed)
    return SpikeLM(97, D=64, layers=2, heads=2, dk=32, dv=32, neurons=48, dtype=dtype, **kw).to(dev)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_whole_in_pieces_and_token_by_token(dev, form):
    m = model(dev, **form)
    tokens = torch.randint(0, 97, (40, 3), device=dev)
    with torch.no_grad():
        whole, after = m(tokens)
        a, state = m(tokens[:17])
        b, state = m(tokens[17:31], state)
        outs = [m.step(tokens[t], state) for t in range(31, 40)]
        again = m.state(3)
        first = m.step(tokens[0], again)
    got = torch.cat([a, b, torch.stack(outs)])
    # the same recurrences in other orders of fp32 sums; spikes may differ only where a membrane meets its threshold
    assert float((got - whole).norm() / whole.norm()) < 2e-3
    assert float((first - whole[0]).norm() / whole[0].norm()) < 1e-4
    for x, y in zip(after, state):
        for s, t in zip(x, y):
            assert s.shape == t.shape and s.dtype == t.dtype
        assert float((x[0] - y[0]).norm() / x[0].norm()) < 2e-3
        if form.get("rotary"):
            assert x[2].tolist() == y[2].tolist() == [40, 40, 40]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_training_on_tokens(dev, form, dtype):
    """Every parameter gets a finite gradient that is not all zero, twice the same bits."""
    m = model(dev, seed=1, dtype=dtype, **form)
    tokens = torch.randint(0, 97, (30, 2), device=dev)
    targets = tokens.roll(-1, 0).clone()
    targets[-1] = -1
    grads = []
    for _ in range(2):
        m.zero_grad(set_to_none=True)
        m.likelihood_loss(tokens, targets).backward()
        grads.append({n: p.grad.clone() for n, p in m.named_parameters()})
    for n, g in grads[0].items():
        assert bool(g.isfinite().all()) and bool(g.any()), n
        assert torch.equal(g, grads[1][n]), n


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_likelihood_gradient_of_the_table(dev, form):
    """d loss / d logits is (softmax - one-hot) / count: the part of the table's gradient that comes through
    the logits, with the blocks' part taken out by differences of two losses' gradients, is what it sends back."""
    m = model(dev, seed=2, **form)
    tokens = torch.randint(0, 97, (12, 2), device=dev)
    targets = torch.randint(-1, 97, (12, 2), device=dev)
    logits, _ = m(tokens)
    z = logits.detach().requires_grad_(True)
    from lifscan import hip_lm as LM
    count = int((targets >= 0).sum())
    (-LM.token_logprobs(z, targets)[0].sum() / count).backward()
    p = z.detach().double().softmax(-1)
    there = (targets >= 0).double()[..., None]
    want = (p - torch.nn.functional.one_hot(targets.clamp(min=0), 97)) * there / count
    assert float((z.grad.double() - want).abs().max()) < 1e-6
    (got,) = torch.autograd.grad(m.likelihood_loss(tokens, targets), m.table)
    (ref,) = torch.autograd.grad(logits, m.table, z.grad)
    assert float((got - ref).norm() / ref.norm()) < 1e-5


def test_scores(dev):
    m = model(dev, seed=3, rotary=True)
    tokens = torch.randint(0, 97, (20, 2), device=dev)
    targets = torch.randint(-1, 97, (20, 2), device=dev)
    with torch.no_grad():
        logits, _ = m(tokens)
        logp, entropy, top, ids = m.score(tokens, targets, temperature=0.8, top=4)
    lp = (logits.double() / 0.8).log_softmax(-1)
    want = lp.gather(-1, targets.clamp(min=0)[..., None])[..., 0] * (targets >= 0)
    assert float((logp - want).abs().max()) < 1e-5 and float((entropy + (lp.exp() * lp).sum(-1)).abs().max()) < 1e-5
    assert torch.equal(ids[..., 0], logits.argmax(-1)) and float((top - lp.gather(-1, ids)).abs().max()) < 1e-5
    assert logp.shape == (20, 2) and ids.shape == (20, 2, 4)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_no_tokens_and_wrong_states(dev, form):
    m = model(dev, **form)
    with torch.no_grad():
        logits, state = m(torch.zeros(0, 3, dtype=torch.int64, device=dev))
        assert logits.shape == (0, 3, 97)
        tok = torch.randint(0, 97, (3,), device=dev)
        assert torch.equal(m.step(tok, state), m.step(tok, m.state(3)))
        for i in range(len(m.state(3)[0])):
            bad = [list(s) for s in m.state(3)]
            bad[1][i] = bad[1][i][:1]
            with pytest.raises(ValueError):
                m.step(tok, [tuple(s) for s in bad])
            bad[1][i] = None
            with pytest.raises(ValueError):
                m(tok[None], [tuple(s) for s in bad])
        with pytest.raises(ValueError):
            m.step(tok, [s[:1] for s in m.state(3)])


def test_decoding_in_a_graph(dev):
    """Steps captured and replayed between eager work: the state advances as eagerly."""
    for form in FORMS[:2]:
        m = model(dev, seed=4, **form)
        tokens = torch.randint(0, 97, (6, 2), device=dev)
        with torch.no_grad():
            eager = m.state(2)
            want = [m.step(tokens[t], eager) for t in range(6)]
            held, tok = m.state(2), tokens[0].clone()

            def one():
                state = list(held)
                out = m.step(tok, state)
                for old, new in zip(held, state):
                    for a, b in zip(old, new):
                        if a is not b:
                            a.copy_(b)
                return out

            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                one()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = one()
            for s in held:
                for t in s:
                    t.zero_()
            for t in range(6):
                tok.copy_(tokens[t])
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want[t])
