"""LUTTransformer with norms, gates, residual scales and dropout masks from a counter: each join against its 64-bit statement on the
tensors that it met in the model, forward and backward."""
import pytest
import torch

import residual_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def model(**more):
    from spiky_b200.lut_layer import SynapseMeta
    from spiky_b200.lut_transformer import LUTTransformer

    args = dict(vocab_size=50, embedding_dim=32, context_size=8, positional_dim=2, num_layers=2, num_heads=2, n_detectors=4,
                n_anchors_per_detector=4, concatenation_product=False, seed=7, device=DEV,
                synapse_meta=SynapseMeta(min_weight=-1.0, max_weight=1.0, initial_noise_level=0.2, initial_weight=-0.1))
    args.update(more)
    return LUTTransformer(**args)


def tokens(B=3, S=8):
    return torch.randint(0, 50, (B, S), generator=torch.Generator().manual_seed(1)).to(DEV)


@pytest.mark.parametrize("opts", [
    dict(norm="rms"), dict(norm="layer", norm_after=True, gated=True, skip_scale=0.875, branch_scale=0.5, dropout=0.2, counter_dropout=True),
    dict(dropout=0.3, counter_dropout=True, dropout_seed=5), dict(gated=True, no_ffn=True, concatenation_product=True),
    dict(norm="layer", embedding_dim=(4, 9), dropout=0.1, counter_dropout=True, concatenation_product=True)])
def test_joins_of_a_model(opts):
    m = model(**opts).train()
    with torch.no_grad():
        for name, p in m.named_parameters():
            if "_join" in name or "first_norm" in name:
                p.add_(0.1 * torch.randn(p.shape, generator=torch.Generator().manual_seed(len(name))).to(DEV))
    seen = []

    def hook(join, args, out):
        for t in args[:2] + out:
            if t.requires_grad and t.grad_fn is not None:
                t.retain_grad()
        seen.append((join, args, out))

    for name, sub in m.named_modules():
        if name.endswith("_join"):
            sub.register_forward_hook(hook)
    logits = m(tokens())
    logits.backward(torch.randn(logits.shape, generator=torch.Generator().manual_seed(2)).to(DEV))
    assert len(seen) == m._n_dropouts

    def cpu(t):
        return None if t is None else t.detach().cpu().double()

    for k, (join, (x, branch, state, site), (h, y)) in enumerate(seen):
        assert site == k
        kept = None
        if join.dropout:
            kept = ro.keeps(join.dropout, *(int(v) for v in (state[0], state[1] + site)), x.numel()).view(x.shape)
        dh = cpu(h.grad) if k + 1 < len(seen) or join.next_norm is None else None
        want = ro.join64(cpu(x), cpu(branch), join.branch_norm, cpu(join.branch_weight), cpu(join.branch_bias), cpu(join.gate), join.skip_scale,
                         join.branch_scale, kept, ro.drop_scale(join.dropout), join.next_norm, cpu(join.next_weight), cpu(join.next_bias), join.eps,
                         dh, cpu(y.grad) if join.next_norm else None)
        ro.assert_near(h, *want["h"], "h")
        ro.assert_near(branch.grad, *want["df"], "df")
        if join.next_norm:
            ro.assert_near(y, *want["y"], "y")
        if k and join.next_norm:   # (the stream goes on to one join alone: its gradient is that join's; without a norm the block reads it too)
            ro.assert_near(x.grad, *want["dx"], "dx")
        for name, key in (("branch_weight", "daw"), ("branch_bias", "dab"), ("next_weight", "dbw"), ("next_bias", "dbb"), ("gate", "dgate")):
            p = getattr(join, name)
            if p is not None:
                ro.assert_near(p.grad, *want[key], name)
    if m.norm:
        assert m.first_norm.weight.grad.isfinite().all()


def test_norms_with_stored_masks():
    """Norms beside torch's own dropout: the modules are called, and evaluation draws nothing."""
    m = model(norm="rms", dropout=0.3).train()
    assert not torch.equal(m(tokens()), m(tokens()))
    m(tokens()).sum().backward()
    assert all(p.grad.isfinite().all() for n, p in m.named_parameters() if "_join" in n or "first_norm" in n)
    m.eval()
    assert torch.equal(m(tokens()), m(tokens()))


def test_models_pickled_before_the_options():
    m = model().eval()
    for name in ("norm", "norm_after", "gated", "counter_dropout", "_joined", "_n_dropouts"):
        del m.__dict__[name]
    assert torch.equal(m(tokens()), m(tokens()))


def test_plain_model_is_what_it_was():
    """Without options the sum is torch's, no buffer and no parameter is added; counter dropout in evaluation mode changes nothing."""
    plain, counted = model(dropout=0.5), model(dropout=0.5, counter_dropout=True)
    assert not any("join" in k or "norm" in k or "dropout" in k for k in plain.state_dict())
    assert [k for k in counted.state_dict() if k not in plain.state_dict()] == ["dropout_state"]
    counted.load_state_dict(plain.state_dict(), strict=False)   # (the seed is that of anchors and embeddings)
    assert torch.equal(plain.eval()(tokens()), counted.eval()(tokens()))
    assert counted.dropout_state.tolist() == [7, 0]


@pytest.mark.parametrize("batch_norm", [False, True])
def test_counter_dropout_is_replayed_from_a_checkpoint(batch_norm):
    m = model(dropout=0.4, counter_dropout=True, use_batch_norm=batch_norm).train()
    saved = {k: v.clone() for k, v in m.state_dict().items()}
    one, two = m(tokens()), m(tokens())
    assert not torch.equal(one, two) and m.dropout_state.tolist() == [7, 8]
    m.load_state_dict(saved)
    assert torch.equal(m(tokens()), one)


def test_training_steps_captured():
    """Training steps replayed from a graph are those run one by one."""
    tok = tokens()
    dl = torch.randn(3, 8, 50, generator=torch.Generator().manual_seed(3)).to(DEV)

    def step(m):
        params = [p for p in m.parameters() if p.requires_grad]
        return torch.autograd.grad(m(tok), params, dl)

    opts = dict(norm="rms", gated=True, dropout=0.3, counter_dropout=True)
    m = model(**opts).train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [[g.clone() for g in step(m)] for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    n = model(**opts).train()
    n.load_state_dict(m.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(n)
    n.dropout_state.copy_(torch.tensor([7, 0]))
    for want in eager:
        graph.replay()
        for a, b in zip(got, want):   # (table gradients are summed by atomics)
            assert (a - b).abs().max() <= 1e-5 * b.abs().max() + 1e-12
    assert torch.equal(n.dropout_state, m.dropout_state)


def test_refusals():
    for bad in (dict(norm="batch"), dict(norm_after=True), dict(use_batch_norm=True, norm="rms"), dict(use_batch_norm=True, gated=True),
                dict(use_batch_norm=True, branch_scale=0.5), dict(dropout_seed=3)):
        with pytest.raises(ValueError):
            model(**bad)
