"""Dropout against its definition: the generator against known words and a numpy form, the
values to one rounding (u of the result, and float32's 2^-23 for the scale and the sum)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from deformops_amd.backends.eager.dropout import kept_elements
from deformops_amd.core.errors import NoBackendError
from deformops_amd.registry import Backend, dropout

F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
IDS = {F32: "f32", F16: "f16", BF16: "bf16", F64: "f64"}
BACKENDS = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="gpu", marks=pytest.mark.gpu)]


def on(device: str) -> str:
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return device


def philox(counter: int, offset: int, seed: int) -> list[int]:
    """Philox4x32-7 on Python integers."""
    word = 2**32
    c = [counter % word, counter // word, offset % word, offset // word]
    key = [seed % word, seed // word]
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b // word ^ c[1] ^ key[0], b % word, a // word ^ c[3] ^ key[1], a % word]
        key = [(key[0] + 0x9E3779B9) % word, (key[1] + 0xBB67AE85) % word]
    return c


def keep_of(n: int, p: float, seed: int, offset: int) -> np.ndarray:
    words = [w for block in range((n + 3) // 4) for w in philox(block, offset, seed)][:n]
    return np.array(words, dtype=np.uint64) >= min(round(p * 2**32), 2**32 - 1)


def test_the_generator_gives_the_published_words():
    """The known answers of Philox4x32 with 7 rounds for counter and key zero."""
    assert philox(0, 0, 0) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    kept = kept_elements(4, 0x4F121F81 / 2**32, torch.tensor(0), 0)
    assert kept.tolist() == [True, False, True, True]
    assert not kept_elements(4, (0x4F121F81 + 1) / 2**32, torch.tensor(0), 0)[2]


SEEDS = [(0, 0), (1, 2**40 + 3), (2**63 - 1, 2**63 - 1), (0x123456789ABCDEF, 7)]


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS.get)
@pytest.mark.parametrize("residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("shape", [(1,), (3, 5), (7, 1, 33), (64, 32), (1, 1027)], ids=str)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_values_and_gradients(device, shape, residual, dtype, p):
    g = torch.Generator().manual_seed(11)
    x, r, grad = (torch.randn(shape, generator=g, dtype=F64).to(dtype).to(on(device)) for _ in range(3))
    seed, offset = SEEDS[len(shape) % 4]
    leaves = [x.requires_grad_()] + ([r.requires_grad_()] if residual else [])
    out = dropout(x, p, seed=seed, offset=offset, residual=r if residual else None)
    grads = torch.autograd.grad(out, leaves, grad)
    keep = torch.from_numpy(keep_of(x.numel(), p, seed, offset) & (p < 1)).view(shape).double()
    factor = keep / (1 - p) if p < 1 else keep
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u
    cpu = [t.detach().cpu().double() for t in (x, r, grad)]
    wanted = cpu[0] * factor
    spread = wanted.abs() * 2.0**-23 + (wanted.abs() + cpu[1].abs()) * 2.0**-23
    wanted = wanted + cpu[1] if residual else wanted
    for got, value, err in ((out, wanted, spread), (grads[0], cpu[2] * factor, (cpu[2] * factor).abs() * 2.0**-23)):
        assert got.dtype == dtype
        off = (got.detach().cpu().double() - value).abs()
        assert (off <= err + u * (value.abs() + err) + tiny).all()
    if not residual:
        assert (out == 0).cpu().eq(keep == 0).all() or (x == 0).any()
    else:
        assert torch.equal(grads[1], grad)


@pytest.mark.parametrize("device", BACKENDS)
def test_dropped_values_leave_nothing(device):
    x = torch.full((1000,), math.nan, device=on(device))
    r = torch.ones(1000, device=device)
    out = dropout(x, 0.5, seed=5, residual=r)
    keep = torch.from_numpy(keep_of(1000, 0.5, 5, 0)).to(device)
    assert out[keep].isnan().all() and out[~keep].eq(1).all()
    assert dropout(x, 1.0, seed=5).eq(0).all()


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=IDS.get)
def test_the_mask_follows_the_logical_order(device, dtype):
    x = torch.randn(30, 50, device=on(device)).to(dtype)
    expected = dropout(x, 0.3, seed=9)
    odd = torch.empty(1501, dtype=dtype, device=device)[1:].view(30, 50).copy_(x)
    for other in (x.t().contiguous().t(), torch.stack([x, x], -1)[..., 0], odd):
        assert torch.equal(dropout(other, 0.3, seed=9), expected)
        assert torch.equal(dropout(x, 0.3, seed=9, residual=other), dropout(x, 0.3, seed=9, residual=x))
    out = dropout(torch.ones(1, device=device).expand(40), 0.5, seed=1)
    assert torch.equal(out, dropout(torch.ones(40, device=device), 0.5, seed=1))


def test_the_share_of_dropped_elements():
    """Of n elements about p n: within 5 standard deviations."""
    n = 2**18
    for p in (0.1, 0.5):
        dropped = int((dropout(torch.ones(n), p, seed=17, offset=3) == 0).sum())
        assert abs(dropped - p * n) < 5 * (n * p * (1 - p)) ** 0.5


@pytest.mark.parametrize("device", BACKENDS)
def test_a_seed_in_memory(device):
    x = torch.randn(77, 5, device=on(device), requires_grad=True)
    for seed in (0, 123456789012345, 2**63 - 1):
        at = torch.tensor([seed], device=device)
        out = dropout(x, 0.4, seed=at, offset=2)
        assert torch.equal(out, dropout(x, 0.4, seed=seed, offset=2))
        assert torch.equal(torch.autograd.grad(out.sum(), x)[0], torch.autograd.grad(
            dropout(x, 0.4, seed=seed, offset=2).sum(), x)[0])
    if device == "cuda":  # the CPU's graph keeps the mask instead
        out = dropout(x, 0.4, seed=at)
        at.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.sum().backward()


@pytest.mark.parametrize("device", BACKENDS)
def test_empty_calls(device):
    x = torch.zeros(0, 3, device=on(device), requires_grad=True)
    out = dropout(x, 0.5, seed=1, residual=x)
    assert out.shape == (0, 3)
    out.sum().backward()


ONE = torch.ones(2, 3)
REFUSALS = {
    "p": (((ONE, 1.5), {"seed": 1}), ValueError, "p must"),
    "p nan": (((ONE, math.nan), {"seed": 1}), ValueError, "p must"),
    "p type": (((ONE, "0.5"), {"seed": 1}), TypeError, "p must"),
    "integers": (((ONE.int(), 0.5), {"seed": 1}), ValueError, "floating"),
    "no seed": (((ONE, 0.5), {}), TypeError, "seed"),
    "seed sign": (((ONE, 0.5), {"seed": -1}), ValueError, "seed"),
    "seed size": (((ONE, 0.5), {"seed": 2**63}), ValueError, "seed"),
    "seed type": (((ONE, 0.5), {"seed": 1.0}), TypeError, "seed"),
    "seed tensor": (((ONE, 0.5), {"seed": torch.ones(2, dtype=torch.int64)}), ValueError, "seed"),
    "seed tensor dtype": (((ONE, 0.5), {"seed": torch.ones(1, dtype=torch.int32)}), ValueError, "seed"),
    "offset": (((ONE, 0.5), {"seed": 1, "offset": -1}), ValueError, "offset"),
    "offset type": (((ONE, 0.5), {"seed": 1, "offset": 0.5}), TypeError, "offset"),
    "residual size": (((ONE, 0.5), {"seed": 1, "residual": torch.ones(3)}), ValueError, "residual"),
    "residual dtype": (((ONE, 0.5), {"seed": 1, "residual": ONE.half()}), ValueError, "residual"),
    "device": (((ONE, 0.5), {"seed": 1, "residual": torch.ones(2, 3, device="meta")}), ValueError, "device"),
    "unknown": (((ONE, 0.5), {"seed": 1, "inplace": True}), TypeError, "unexpected"),
}


@pytest.mark.parametrize("device", BACKENDS)
@pytest.mark.parametrize("name", REFUSALS)
def test_refusals(device, name):
    (args, options), error, words = REFUSALS[name]
    on(device)

    def moved(t):
        return t.to(device) if isinstance(t, torch.Tensor) and t.device.type != "meta" else t

    with pytest.raises(error, match=words):
        dropout(*map(moved, args), **{k: moved(v) for k, v in options.items()})


@pytest.mark.gpu
def test_gpu_calls_that_no_kernel_takes(device):
    with pytest.raises(NoBackendError):
        dropout(torch.ones(3, dtype=F64, device=device), 0.5, seed=1)
    assert dropout.resolve(ONE.to(device), 0.5, seed=1).backend is Backend.HIP


@pytest.mark.parametrize("device", BACKENDS)
def test_vmap_tracing_and_the_public_operator(device):
    x = torch.randn(6, 7, device=on(device), requires_grad=True)
    r = torch.randn(6, 7, device=device, requires_grad=True)
    expected = dropout(x, 0.5, seed=3, offset=4, residual=r)
    with pytest.raises(RuntimeError, match="vmap"):
        torch.vmap(lambda a: dropout(a, 0.5, seed=3))(x)
    torch.testing.assert_close(torch.ops.deformops.dropout(x, 0.5, 3, None, 4, r), expected)
    compiled = torch.compile(lambda a, b: dropout(a, 0.5, seed=3, offset=4, residual=b), backend="aot_eager",
                             fullgraph=True)(x, r)
    torch.testing.assert_close(compiled, expected)
    for a, b in zip(torch.autograd.grad(compiled.sum(), (x, r)), torch.autograd.grad(expected.sum(), (x, r))):
        torch.testing.assert_close(a, b)


@pytest.mark.gpu
def test_a_graph_reads_the_seed_at_every_replay(device):
    x = torch.randn(300, 64, device=device, requires_grad=True)
    seed = torch.zeros(1, dtype=torch.int64, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def call(at):
        out = dropout(x, 0.3, seed=at, residual=x)
        return out.detach(), torch.autograd.grad(out.sum(), x)[0]

    with torch.cuda.stream(side):
        call(seed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = call(seed)
    for turn in (5, 5, 2**50):
        seed.fill_(turn)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, call(turn)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_devices_drop_the_same_elements(device):
    x = torch.ones(2**20 + 3, device=device)
    out = dropout(x, 0.25, seed=2**61 + 5, offset=2**33)
    assert torch.equal(out.cpu(), dropout(x.cpu(), 0.25, seed=2**61 + 5, offset=2**33))


@pytest.mark.gpu
def test_counters_past_32_bits(device):
    """The last elements of a tensor of more than 2^32."""
    n = 2**32 + 2**20 + 9
    out = dropout(torch.ones((), dtype=BF16, device=device).expand(n).contiguous(), 0.5, seed=3)
    first = (n - 8) // 4
    words = [w for block in range(first, first + 3) for w in philox(block, 0, 3)][:n - 4 * first]
    assert (out[4 * first:] != 0).tolist() == [w >= 2**31 for w in words]
