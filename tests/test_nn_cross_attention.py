"""The operators beside MSDA as a decoder runs them together: the cross attention layer, the
dropped residual of the MSDA layer, and Mask2Former's decoder.

The layer is compared with its own parts in 64 bits. With n products in a row, float32
results are held to 1e-5 and gradients to 1e-4 of the largest element (the sums have at
most 512 terms of 2^-24 each, through four products), 16-bit ones to 4 u and 8 u: a
projection, the turn, the attention and the output's projection round once each, a
gradient passes them twice.
"""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

from deformops_amd.nn import CrossAttention, MultiScaleDeformAttn2d
from deformops_amd.registry import dropout, rotary
from tests.test_dropout import keep_of
from tests.test_rotary import reference as turned

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}
BACKENDS = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="gpu", marks=pytest.mark.gpu)]


def on(device: str) -> str:
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return device


class Plain(nn.Module):
    """The layer in elementary operations, in 64 bits on the CPU."""

    def __init__(self, layer: CrossAttention) -> None:
        super().__init__()
        self.layer = copy.deepcopy(layer).cpu().double()
        self.frequencies = layer.frequencies.cpu().double() if layer.rotary_sections else None

    def turn(self, x, positions):
        if positions is None:
            return x
        axis = [a for a, n in enumerate(self.layer.rotary_sections) for _ in range(n)]
        angle = (positions.cpu().double()[..., axis] * self.frequencies).unsqueeze(-2)
        R = len(axis)
        a, b = x[..., :R], x[..., R:2 * R]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., 2 * R:]], -1)

    def forward(self, q, context, positions, places, mask, lengths, residual, seed):
        m = self.layer
        (B, Q, _), S = q.shape, context.shape[1]
        query = self.turn(m.proj_query(q).view(B, Q, m.num_heads, m.head_dim), positions)
        shape, group = (B, S, m.num_key_heads, m.head_dim), m.num_heads // m.num_key_heads
        key = self.turn(m.proj_key(context).view(shape), places).repeat_interleave(group, 2)
        value = m.proj_value(context).view(shape).repeat_interleave(group, 2)
        scores = torch.einsum("bqhd,bshd->bhqs", query, key) / m.head_dim**0.5
        off = torch.arange(S) >= lengths.cpu()[:, None, None, None]
        off = off | ~mask.cpu()
        weights = torch.softmax(scores.masked_fill(off, -1e300), -1).masked_fill(off, 0.0)
        out = m.proj_output(torch.einsum("bhqs,bshd->bqhd", weights, value).reshape(B, Q, -1))
        keep = torch.from_numpy(keep_of(out.numel(), m.dropout, seed, 0)).view(out.shape)
        return out * keep / (1 - m.dropout) + residual


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("axes", [0, 3])
def test_the_operators_together(device, axes, dtype):
    """Projections, rotary positions, masked attention over padded states with shared heads,
    dropout and the residual: outputs and every gradient."""
    torch.manual_seed(3)
    layer = CrossAttention(64, 48, num_heads=4, num_key_heads=2, rotary_sections=(2, 3, 3) if axes else None, dropout=0.2)
    layer = layer.to(on(device), dtype)
    B, Q, S = 2, 30, 75
    g = torch.Generator().manual_seed(1)
    inputs = [torch.randn(s, generator=g, dtype=F64).to(dtype).to(device).requires_grad_()
              for s in ((B, Q, 64), (B, S, 48), (B, Q, 64))]
    grad = torch.randn(B, Q, 64, generator=g, dtype=F64).to(dtype).to(device)
    positions, places = (torch.randint(0, 500, (n, 3), generator=g).to(device) if axes else None for n in (Q, S))
    mask = torch.rand(B, 1, Q, S, generator=g) < 0.7
    mask[:, :, ::9] = False
    mask, lengths = mask.to(device), torch.tensor([75, 40], device=device)
    out = layer(*inputs[:2], positions=positions, context_positions=places, mask=mask, key_lengths=lengths,
                residual=inputs[2], seed=12)
    grads = torch.autograd.grad(out, [*inputs, *layer.parameters()], grad)

    plain = Plain(layer)
    wide = [t.detach().cpu().double().requires_grad_() for t in inputs]
    expected = plain(*wide[:2], positions, places, mask, lengths, wide[2], 12)
    wanted = torch.autograd.grad(expected, [*wide, *plain.layer.parameters()], grad.cpu().double())
    u = torch.finfo(dtype).eps / 2
    names = ["q", "context", "residual", *(name for name, _ in layer.named_parameters())]
    # A score's gradients add up to 0 along a row's states, so without a turn the gradient of
    # the keys' bias, the sum of dk over all states, is 0 by definition: what is left of its
    # terms is their rounding. Its terms are those of the keys' weight (times states of size
    # 1), whose gradient is the measure.
    sizes = {name: e.abs().max() for name, e in zip(names, wanted)}
    sizes["proj_key.bias"] = max(sizes["proj_key.bias"], sizes["proj_key.weight"])
    for bound, pairs in ((1e-5 if dtype == F32 else 4 * u, [(out, expected, expected.detach().abs().max())]),
                         (1e-4 if dtype == F32 else 8 * u,
                          [(a, e, sizes[name]) for a, e, name in zip(grads, wanted, names)])):
        for a, e, size in pairs:
            assert a.shape == e.shape
            assert (a.detach().cpu().double() - e.detach()).abs().max() <= bound * size


@pytest.mark.parametrize("device", BACKENDS)
def test_a_decoders_steps_over_kept_states(device):
    """Tokens one at a time over states made once give what all of them give together."""
    torch.manual_seed(0)
    layer = CrossAttention(128, num_heads=4, num_key_heads=1, rotary_sections=(4, 4)).to(on(device)).eval()
    q, context = torch.randn(3, 7, 128, device=device), torch.randn(3, 500, 128, device=device)
    positions, places = torch.rand(7, 2, device=device) * 50, torch.rand(3, 500, 2, device=device) * 50
    lengths = torch.tensor([500, 0, 123], device=device)
    with torch.no_grad():
        whole = layer(q, context, positions=positions, context_positions=places, key_lengths=lengths)
        states = layer.states(context, places)
        for i in range(7):
            one = layer(q[:, i:i + 1], states, positions=positions[i:i + 1], key_lengths=lengths)
            torch.testing.assert_close(one, whole[:, i:i + 1], rtol=1e-5, atol=1e-5)


def test_layer_arguments():
    for options in ({"num_heads": 3}, {"num_heads": 0}, {"num_heads": 4, "num_key_heads": 3},
                    {"num_heads": 4, "dropout": 1.5}, {"num_heads": 4, "rotary_sections": (5, 4)},
                    {"num_heads": 4, "rotary_sections": (5, -4)}):
        with pytest.raises(ValueError):
            CrossAttention(64, **options)
    layer = CrossAttention(32, num_heads=2, rotary_sections=(4,), dropout=0.5)
    q, places = torch.randn(1, 3, 32), torch.arange(3)[:, None]
    with pytest.raises(ValueError, match="positions are needed"):
        layer(q, q, context_positions=places)
    with pytest.raises(ValueError, match="context_positions"):
        layer(q, layer.states(q, places), positions=places, context_positions=places)
    with pytest.raises(ValueError, match="without rotary_sections"):
        CrossAttention(32, num_heads=2)(q, q, positions=places)
    assert "frequencies" not in layer.state_dict() and "dropout=0.5" in repr(layer)


def test_dropout_is_for_training_and_draws_its_seed():
    layer = CrossAttention(32, num_heads=2, dropout=0.5)
    q = torch.randn(1, 30, 32)
    torch.manual_seed(1)
    first = layer(q, q)
    torch.manual_seed(1)
    assert torch.equal(layer(q, q), first) and not torch.equal(layer(q, q), first)
    assert torch.equal(layer(q, q, seed=5), layer(q, q, seed=torch.tensor(5)))
    layer.eval()
    assert torch.equal(layer(q, q), layer(q, q)) and layer(q, q).ne(0).all()
    torch.testing.assert_close(layer(q, q, residual=q), layer(q, q) + q)


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("training", [True, False], ids=["train", "eval"])
def test_a_residual_of_another_dtype(device, training):
    """Under autocast the output is narrow and the residual is not: both are added in the wider dtype."""
    torch.manual_seed(3)
    layer = CrossAttention(32, num_heads=2, dropout=0.25).to(on(device)).train(training)
    q = torch.randn(2, 9, 32, device=device)
    residual = torch.randn(2, 9, 32, device=device, requires_grad=True)
    with torch.autocast(device, dtype=BF16):
        out = layer(q, q, residual=residual, seed=4)
        bare = layer.eval()(q, q)
    assert out.dtype == F32 and bare.dtype == BF16
    wide = bare.float()
    expected = dropout(wide, 0.25, seed=4, residual=residual) if training else wide + residual
    assert torch.equal(out, expected)
    grads = torch.autograd.grad(out.sum(), [residual, layer.proj_output.weight])
    assert grads[0].eq(1).all() and grads[1].isfinite().all() and grads[1].ne(0).any()


def test_an_msda_layer_that_was_pickled_without_dropout():
    layer = MultiScaleDeformAttn2d(32, num_heads=4, num_levels=1)
    inputs = (torch.randn(1, 3, 32), torch.rand(1, 3, 1, 2), torch.randn(1, 12, 32), torch.tensor([[4, 3]]),
              torch.tensor([0]))
    expected = layer(*inputs)
    layer.__dict__.pop("dropout", None)
    assert torch.equal(layer(*inputs), expected) and "dropout" not in repr(layer)


@pytest.mark.gpu
def test_a_captured_layer_needs_a_seed_in_memory(device):
    layer = CrossAttention(32, num_heads=2, dropout=0.5).to(device)
    q = torch.randn(1, 3, 32, device=device)
    seed = torch.ones(1, dtype=torch.int64, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        layer(q, q, seed=seed)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="needs seed"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            layer(q, q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer(q, q, seed=seed)
        for n in (4, 9, 4):
            seed.fill_(n)
            graph.replay()
            torch.cuda.synchronize()
            torch.testing.assert_close(out, layer(q, q, seed=n))


@pytest.mark.parametrize("device", BACKENDS)
def test_the_msda_layers_dropped_residual(device):
    torch.manual_seed(2)
    layer = MultiScaleDeformAttn2d(32, num_heads=4, num_levels=2, dropout=0.3).to(on(device))
    shapes, starts = torch.tensor([[6, 5], [3, 2]], device=device), torch.tensor([0, 30], device=device)
    q, v = torch.randn(2, 11, 32, device=device), torch.randn(2, 36, 32, device=device)
    p, r = torch.rand(2, 11, 2, 2, device=device), torch.randn(2, 11, 32, device=device, requires_grad=True)
    layer.eval()
    bare = layer(q, p, v, shapes, starts)
    torch.testing.assert_close(layer(q, p, v, shapes, starts, residual=r), bare + r)
    layer.train()
    out = layer(q, p, v, shapes, starts, residual=r, seed=8)
    torch.testing.assert_close(out, dropout(bare, 0.3, seed=8, residual=r))
    grads = torch.autograd.grad(out.sum(), [r, layer.proj_output.bias])
    keep = torch.from_numpy(keep_of(out.numel(), 0.3, 8, 0)).view(-1, 32).sum(0).float() / 0.7
    assert grads[0].eq(1).all()
    torch.testing.assert_close(grads[1].cpu(), keep)
    assert MultiScaleDeformAttn2d(32, num_heads=4, num_levels=2).dropout == 0.0
    with pytest.raises(ValueError):
        MultiScaleDeformAttn2d(32, num_heads=4, num_levels=2, dropout=-0.1)


@pytest.mark.parametrize("device", BACKENDS)
def test_rotary_scores_depend_on_differences_of_places(device):
    """q at p and k at s score as q at p + t and k at s + t, on every axis at once."""
    q, k = torch.randn(1, 20, 2, 32, device=on(device)), torch.randn(1, 20, 2, 32, device=device)
    places = torch.randint(0, 100, (20, 2), device=device)
    layer = CrossAttention(64, num_heads=2, rotary_sections=(8, 8)).to(device)

    def scores(shift):
        a, b = (rotary(t, places + torch.tensor(shift, device=device), layer.frequencies, sections=(8, 8)) for t in (q, k))
        return torch.einsum("bqhd,bshd->bhqs", a, b)

    torch.testing.assert_close(scores((0, 0)), scores((1000, -77)), rtol=1e-4, atol=1e-4)
    assert turned(q, places, layer.frequencies, (8, 8), False)[0].shape == q.shape


# Mask2Former's decoder.


def masked_attention(device, kind, dropout_p=0.0):
    torch.manual_seed(4)
    module = nn.MultiheadAttention(32, 4, dropout_p).to(device)
    with torch.no_grad():
        module.in_proj_bias.normal_()
    g = torch.Generator().manual_seed(5)
    query, key, value = (torch.randn(n, 2, 32, generator=g).to(device).requires_grad_() for n in (9, 40, 40))
    mask = padding = None
    if kind == "bool":
        mask = torch.rand(8, 9, 40, generator=g) < 0.5
    elif kind == "float":
        mask = torch.randn(8, 9, 40, generator=g)
    elif kind == "rows":
        mask = torch.rand(9, 40, generator=g) < 0.5
    elif kind == "padded":
        mask = torch.rand(8, 9, 40, generator=g) < 0.5
        padding = torch.zeros(2, 40, dtype=torch.bool)
        padding[1, 30:] = True
    return module, (query, key, value), *(None if t is None else t.to(device) for t in (mask, padding))


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("kind", ["none", "bool", "float", "rows", "padded"])
def test_masked_attention_matches_the_module_it_replaces(device, kind):
    integ = pytest.importorskip("deformops_amd.integrations.transformers")
    old, inputs, mask, padding = masked_attention(on(device), kind)
    new = integ.Mask2FormerMaskedCrossAttention(copy.deepcopy(old))
    runs = []
    for module in (old, new):
        extra = {} if module is new else {"need_weights": False}
        out, weights = module(*inputs, attn_mask=mask, key_padding_mask=padding, **extra)
        grads = torch.autograd.grad(out.pow(2).sum(), [*inputs, *module.parameters()])
        assert weights is None
        runs.append((out, grads))
    torch.testing.assert_close(runs[0][0], runs[1][0], rtol=1e-5, atol=1e-5)
    assert [n for n, _ in old.named_parameters()] == [n for n, _ in new.named_parameters()]
    for a, e in zip(runs[1][1], runs[0][1]):
        torch.testing.assert_close(a, e, rtol=1e-4, atol=1e-4)


def three_layers(model: nn.Module) -> nn.Module:
    """The tiny model, whose configuration leaves its decoder without layers, with three."""
    integ = pytest.importorskip("deformops_amd.integrations.transformers")
    decoder = next(m for m in model.modules() if isinstance(m, integ._m2f.Mask2FormerMaskedAttentionDecoder))
    decoder.layers = nn.ModuleList(integ._m2f.Mask2FormerMaskedAttentionDecoderLayer(decoder.config) for _ in range(3))
    return model.eval()


@pytest.mark.parametrize("device", BACKENDS)
def test_a_patched_decoder_matches_upstream(device):
    integ = pytest.importorskip("deformops_amd.integrations.transformers")
    from tests.test_integrations_transformers import generic_sampling, tiny_mask2former  # noqa: PLC0415

    torch.manual_seed(0)
    upstream = three_layers(generic_sampling(tiny_mask2former())).to(on(device))
    patched = integ.patch(copy.deepcopy(upstream), decoder=True)
    kinds = [type(m) for m in patched.modules()]
    layers = sum(isinstance(m, integ._m2f.Mask2FormerMaskedAttentionDecoderLayer) for m in patched.modules())
    assert kinds.count(integ.Mask2FormerMaskedCrossAttention) == layers == 3
    assert kinds.count(integ.Mask2FormerPixelDecoderEncoderMultiscaleDeformableAttention) == 2
    assert set(patched.state_dict()) == set(upstream.state_dict())
    image = torch.randn(1, 3, 64, 64, generator=torch.Generator().manual_seed(1)).to(device)
    with torch.no_grad():
        expected, actual = upstream(image), patched(image)
    torch.testing.assert_close(actual.class_queries_logits, expected.class_queries_logits, rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(actual.masks_queries_logits, expected.masks_queries_logits, rtol=1e-3, atol=1e-3)


def test_what_the_decoders_patch_leaves_and_refuses():
    integ = pytest.importorskip("deformops_amd.integrations.transformers")
    from tests.test_integrations_transformers import RecordingOracleBackend, tiny_mask2former  # noqa: PLC0415

    model = integ.patch(tiny_mask2former())
    assert not any(isinstance(m, integ.Mask2FormerMaskedCrossAttention) for m in model.modules())
    with pytest.raises(TypeError, match="Backend member"):
        integ.patch(model, decoder=True, backend=RecordingOracleBackend())
    with pytest.raises(ValueError, match="attention weights"):
        integ.Mask2FormerMaskedCrossAttention(masked_attention("cpu", "none", 0.1)[0])
    with pytest.raises(ValueError, match="sequence first"):
        integ.Mask2FormerMaskedCrossAttention(nn.MultiheadAttention(32, 4, batch_first=True))
