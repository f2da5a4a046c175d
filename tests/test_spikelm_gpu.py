"""GPU: the spiking language model (lifscan.spikelm), which runs the language-model operators and the
neurons together: a sequence fed whole, in pieces and token by token, and training by distillation."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dev, dtype=torch.float32):
    from lifscan.spikelm import SpikeLM
    torch.manual_seed(0)
    return SpikeLM(200, D=96, layers=2, heads=3, dk=32, dv=48, neurons=128, dtype=dtype).to(dev)


def test_whole_in_pieces_and_token_by_token(dev):
    """The three ways differ in the rounding of their sums (below 1e-5 of the values) as long as no neuron
    comes that close to its threshold: of the 23040 neuron-steps here at a density of the potentials of
    about one per unit a quarter of one would, and the spikes of these seeds agree."""
    model = _model(dev)
    tokens = torch.randint(0, 200, (45, 2), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        whole, _ = model(tokens)
        carried, after = model(tokens, model.state(2))
        first, state = model(tokens[:19], model.state(2))
        second, state = model(tokens[19:40], state)
        last = [model.step(tokens[t], state) for t in range(40, 45)]
    pieces = torch.cat([first, second, torch.stack(last)])
    scale = float(whole.abs().max())
    assert float((carried - whole).abs().max()) < 1e-4 * scale
    assert float((pieces - whole).abs().max()) < 1e-4 * scale
    for (S, u), (S2, u2) in zip(state, after):
        assert float((S - S2).abs().max()) < 1e-4 * float(S.abs().max()) and float((u - u2).abs().max()) < 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_training_by_distillation(dev, dtype):
    model = _model(dev, dtype)
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 200, (33, 4), generator=g).to(dev)
    index = torch.randint(0, 200, (33, 4, 8), generator=g).to(dev)
    values = torch.randn(33, 4, 8, generator=g).to(dev)
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(30):
        opt.zero_grad()
        loss = model.loss(tokens, values, index, temperature=2.0)
        loss.backward()
        for name, p in model.named_parameters():
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0, name
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.7 * losses[0], losses


def test_a_prompt_then_its_next_tokens(dev):
    """The state that forward returns without gradients continues the sequence, token by token or in pieces."""
    model = _model(dev)
    tokens = torch.randint(0, 200, (45, 2), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        whole, _ = model(tokens, model.state(2))
        prompt, state = model(tokens[:30])
        piece, state = model(tokens[30:40], state)
        last = [model.step(tokens[t], state) for t in range(40, 45)]
    pieces = torch.cat([prompt, piece, torch.stack(last)])
    assert float((pieces - whole).abs().max()) < 1e-4 * float(whole.abs().max())


def test_states_that_do_not_continue_a_sequence(dev):
    """Training returns no state; a state that is not whole is refused before any of it is changed; a call with a
    state has no gradients."""
    model = _model(dev)
    tokens = torch.randint(0, 200, (5, 2), generator=torch.Generator().manual_seed(1)).to(dev)
    logits, state = model(tokens)
    assert logits.requires_grad and state is None
    with torch.no_grad():
        _, good = model(tokens, model.state(2))
    S = good[0][0].clone()
    for bad in ([good[0], (good[1][0], None)], good[:1], [good[0], (good[1][0][:1], good[1][1])],
                [good[0], (good[1][0], good[1][1][:-1])], [good[0], None],
                [good[0], (good[1][0].double(), good[1][1])], [good[0], (good[1][0], good[1][1].cpu())]):
        with pytest.raises(ValueError):
            model.step(tokens[0], list(bad))
        with pytest.raises(ValueError):
            model(tokens, list(bad))
    assert torch.equal(S, good[0][0])
    logits, _ = model(tokens, good)
    assert not logits.requires_grad


def test_no_tokens(dev):
    """A sequence without tokens: no logits, the state that it began with, gradients of zero."""
    model = _model(dev)
    none = torch.zeros(0, 2, dtype=torch.int64, device=dev)
    logits, state = model(none)
    assert logits.shape == (0, 2, 200) and state is None
    logits.sum().backward()
    assert all(p.grad is None or bool((p.grad == 0).all()) for p in model.parameters())
    with torch.no_grad():
        logits, state = model(none)
        assert logits.shape == (0, 2, 200) and all(bool((t == 0).all()) for s in state for t in s)
        _, good = model(torch.ones(3, 2, dtype=torch.int64, device=dev))
        _, same = model(none, good)
    for a, b in zip(good, same):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
