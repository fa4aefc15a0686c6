"""Rotary positions against complex products in 64 bits.

Tolerance of one result a cos - b sin: the angle's cosine and sine in float32 are off by
2^-24 for their own rounding, by 2 pi 2^-26 for the fraction's (at most 1/2, kept in
float32: half a step 2^-26) and, on the GPU, by 2^-23 for sinpi and cospi (2 ulp); the two
products and their sum round by 2^-23 (|a| + |b|); the result is rounded once, by u of
its magnitude.
"""

from __future__ import annotations

import math

import pytest
import torch
from torch import Tensor

from deformops_amd.core.errors import NoBackendError
from deformops_amd.registry import Backend, rotary, rotary_frequencies

F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
IDS = {F32: "f32", F16: "f16", BF16: "bf16", F64: "f64"}
BACKENDS = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="gpu", marks=pytest.mark.gpu)]


def on(device: str) -> str:
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return device


def reference(x, positions, frequencies, sections, interleaved, sign=1.0):
    """``(value, bound)`` in 64 bits on the CPU."""
    x, frequencies = x.detach().cpu().double(), frequencies.cpu().double()
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = positions.cpu().double()[..., axis] * frequencies
    turn = torch.polar(torch.ones_like(angle), sign * angle).unsqueeze(-2)
    R = len(axis)
    a = x[..., 0:2 * R:2] if interleaved else x[..., :R]
    b = x[..., 1:2 * R:2] if interleaved else x[..., R:2 * R]
    both = torch.view_as_real(torch.complex(a, b) * turn)
    size = (a.abs() + b.abs()).unsqueeze(-1).expand(both.shape)
    value, spread = x.clone(), torch.zeros_like(x)
    if interleaved:
        value[..., :2 * R], spread[..., :2 * R] = both.flatten(-2), size.flatten(-2)
    else:
        value[..., :2 * R] = both.transpose(-1, -2).flatten(-2)
        spread[..., :2 * R] = size.transpose(-1, -2).flatten(-2)
    return value, spread * (2.0**-24 + math.tau * 2.0**-26 + 2.0**-23 + 2.0**-23)


def assert_turned(actual: Tensor, expected: tuple[Tensor, Tensor]) -> None:
    value, spread = expected
    u = torch.finfo(actual.dtype).eps / 2
    tiny = torch.finfo(actual.dtype).smallest_normal * u
    actual = actual.detach().cpu().double()
    assert actual.shape == value.shape
    over = (actual - value).abs() - (spread + u * (value.abs() + spread) + tiny)
    assert not over.numel() or over.max() <= 0, f"off by {(actual - value).abs().max()} at element {int(over.argmax())}"


def make(B, L, H, D, axes, dtype, device, kind="i64", per_image=True, far=1000):  # noqa: N803
    g = torch.Generator().manual_seed(7)
    x = torch.randn(B, L, H, D, generator=g, dtype=F64).to(dtype).to(device)
    grad = torch.randn(B, L, H, D, generator=g, dtype=F64).to(dtype).to(device)
    shape = (B, L, axes) if per_image else (L, axes)
    positions = torch.randint(-far, far, shape, generator=g)
    if kind.startswith("f"):
        positions = positions + torch.rand(shape, generator=g, dtype=F64)
    positions = positions.to({"i64": torch.int64, "i32": torch.int32, "f32": F32, "f64": F64}[kind])
    return x, positions.to(device), grad


CASES = [  # B, L, H, D, sections
    (1, 1, 1, 2, (1,)),
    (1, 1, 16, 64, (8, 12, 12)),
    (2, 37, 8, 32, (0, 5, 6)),
    (3, 130, 3, 80, (8, 16, 16)),
    (1, 200, 1, 128, (16, 24, 24)),
    (2, 5, 2, 7, (2, 1)),
    (1, 9, 2, 512, (256,)),
    (2, 33, 4, 96, (8, 8)),
    (1, 2000, 8, 64, (16, 16)),
]


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS.get)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])))
def test_turns_and_gradients(device, case, interleaved, dtype):
    B, L, H, D, sections = case
    x, positions, grad = make(B, L, H, D, len(sections), dtype, on(device))
    frequencies = rotary_frequencies(sections, device=device)
    x.requires_grad_()
    out = rotary(x, positions, frequencies, sections=sections, interleaved=interleaved)
    assert out.is_contiguous() and out.dtype == dtype
    assert_turned(out, reference(x, positions, frequencies, sections, interleaved))
    assert_turned(torch.autograd.grad(out, x, grad)[0],
                  reference(grad, positions, frequencies, sections, interleaved, -1.0))


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("kind", ["i64", "i32", "f32", "f64"])
@pytest.mark.parametrize("per_image", [False, True])
def test_positions_of_every_type_and_far_ones(device, kind, per_image):
    x, positions, _ = make(2, 50, 2, 32, 3, F32, on(device), kind, per_image, far=10**6)
    sections = (4, 6, 6)
    frequencies = rotary_frequencies(sections, device=device, shared=True)
    out = rotary(x, positions, frequencies, sections=sections)
    assert_turned(out, reference(x, positions, frequencies, sections, False))
    # strides of their own, and one that serves every image
    wide = torch.stack([positions, positions], -1)[..., 0]
    assert torch.equal(rotary(x, wide, frequencies, sections=sections), out)
    if not per_image:
        assert torch.equal(rotary(x, positions[None], frequencies, sections=sections), out)


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=IDS.get)
def test_layouts_of_x(device, dtype):
    x, positions, _ = make(2, 40, 4, 32, 1, dtype, on(device))
    frequencies = rotary_frequencies((16,), device=device)
    expected = rotary(x, positions, frequencies)
    packed = torch.cat([x, x], -1)[..., 32:]
    odd = torch.empty(x.numel() + 1, dtype=dtype, device=device)[1:].view(x.shape).copy_(x)
    for other in (x.transpose(1, 2).contiguous().transpose(1, 2), packed, odd,
                  x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)):
        assert torch.equal(rotary(other, positions, frequencies), expected)
    one = x[:1, :1].expand(2, 40, 4, 32)
    assert_turned(rotary(one, positions, frequencies), reference(one, positions, frequencies, (16,), False))


@pytest.mark.parametrize("device", BACKENDS)
def test_empty_calls_and_no_pairs(device):
    frequencies = rotary_frequencies((), device=on(device))
    x = torch.randn(2, 3, 2, 8, device=device)
    none = rotary(x, torch.zeros(3, 1, device=device), torch.zeros(0, device=device), sections=(0,))
    assert torch.equal(none, x) and frequencies.numel() == 0
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        y = rotary(torch.zeros(shape, device=device), torch.zeros(shape[1], 1, device=device),
                   rotary_frequencies((4,), device=device))
        assert y.shape == shape


def bad(**changes):
    call = {"x": torch.zeros(2, 3, 2, 8), "positions": torch.zeros(3, 2), "frequencies": torch.ones(4),
            "sections": (2, 2)}
    call.update(changes)
    return call


REFUSALS = {
    "rank": (bad(x=torch.zeros(2, 3, 8)), ValueError, "x must"),
    "integers": (bad(x=torch.zeros(2, 3, 2, 8, dtype=torch.int32)), ValueError, "floating"),
    "tokens": (bad(positions=torch.zeros(4, 2)), ValueError, "positions"),
    "images": (bad(positions=torch.zeros(3, 3, 2)), ValueError, "positions"),
    "positions dtype": (bad(positions=torch.zeros(3, 2, dtype=torch.int16)), ValueError, "positions"),
    "positions gradient": (bad(positions=torch.zeros(3, 2, requires_grad=True)), NotImplementedError, "positions"),
    "frequencies dtype": (bad(frequencies=torch.ones(4, dtype=F64)), ValueError, "frequencies"),
    "frequencies gradient": (bad(frequencies=torch.ones(4, requires_grad=True)), NotImplementedError, "frequencies"),
    "too many": (bad(frequencies=torch.ones(5), sections=(2, 3)), ValueError, "features"),
    "axes": (bad(sections=(4,)), ValueError, "sections"),
    "sum": (bad(sections=(2, 1)), ValueError, "sections"),
    "negative": (bad(sections=(5, -1)), ValueError, "sections"),
    "no sections": (bad(sections=None), ValueError, "sections"),
    "device": (bad(frequencies=torch.ones(4, device="meta")), ValueError, "device"),
}


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("name", REFUSALS)
def test_refusals(device, name):
    call, error, words = REFUSALS[name]
    on(device)
    moved = [t if t.device.type == "meta" else t.detach().to(device).requires_grad_(t.requires_grad)
             for t in (call["x"], call["positions"], call["frequencies"])]
    with pytest.raises(error, match=words):
        rotary(*moved, sections=call["sections"])


def test_call_surface():
    call = bad()
    with pytest.raises(TypeError, match="positionally"):
        rotary(call["x"], call["positions"])
    with pytest.raises(TypeError, match="unexpected"):
        rotary(call["x"], call["positions"], call["frequencies"], base=2)
    assert rotary.resolve(call["x"], call["positions"], call["frequencies"], sections=(2, 2)).backend is Backend.EAGER


@pytest.mark.gpu
def test_gpu_calls_that_no_kernel_takes(device):
    for x, R in ((torch.zeros(1, 1, 1, 8, dtype=F64), 4), (torch.zeros(1, 1, 1, 600), 300),
                 (torch.zeros(1, 1, 2**11, 2**10), 4)):
        with pytest.raises(NoBackendError):
            rotary(x.to(device), torch.zeros(1, 1, device=device), rotary_frequencies((R,), device=device))


@pytest.mark.parametrize("device", BACKENDS)
def test_vmap_tracing_and_the_public_operator(device):
    x, positions, grad = make(6, 5, 2, 16, 2, F32, on(device))
    sections = (3, 4)
    frequencies = rotary_frequencies(sections, device=device)
    x.requires_grad_()
    whole = rotary(x, positions, frequencies, sections=sections)
    expected = torch.autograd.grad(whole, x, grad)[0]
    mapped = torch.vmap(lambda a, p: rotary(a, p, frequencies, sections=sections))(x.view(3, 2, 5, 2, 16),
                                                                                  positions.view(3, 2, 5, 2))
    torch.testing.assert_close(mapped.reshape(whole.shape), whole)
    with pytest.raises(RuntimeError, match="frequencies"):
        torch.vmap(lambda f: rotary(x, positions, f, sections=sections))(torch.stack([frequencies] * 2))
    torch.testing.assert_close(torch.ops.deformops.rotary(x, positions, frequencies, list(sections), False), whole)
    compiled = torch.compile(lambda a: rotary(a, positions, frequencies, sections=sections), backend="aot_eager",
                             fullgraph=True)(x)
    torch.testing.assert_close(compiled, whole)
    torch.testing.assert_close(torch.autograd.grad(compiled, x, grad)[0], expected)


@pytest.mark.gpu
def test_another_stream_and_a_graph(device):
    x, positions, grad = make(2, 300, 8, 64, 3, BF16, device)
    sections = (8, 12, 12)
    frequencies = rotary_frequencies(sections, device=device)
    side = torch.cuda.Stream()
    static = x.clone().requires_grad_()
    side.wait_stream(torch.cuda.current_stream())

    def call(a):
        out = rotary(a, positions, frequencies, sections=sections)
        return out.detach(), torch.autograd.grad(out, a, grad)[0]

    with torch.cuda.stream(side):
        call(static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = call(static)
    for turn in range(3):
        fresh = (x * (turn + 1)).detach().requires_grad_()
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, call(fresh)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_tensor_whose_offsets_pass_32_bits(device):
    L, H, D = 2**17 + 3, 128, 128
    x = torch.zeros(1, L, H, D, dtype=BF16, device=device)
    assert x.numel() > 2**31
    x[:, -2:] = torch.randn(1, 2, H, D, device=device).to(BF16)
    positions = torch.arange(L, device=device)[:, None]
    frequencies = rotary_frequencies((64,), device=device)
    out = rotary(x, positions, frequencies)
    assert_turned(out[:, -2:], reference(x[:, -2:], positions[-2:], frequencies, (64,), False))
