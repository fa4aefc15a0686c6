"""Cross attention, rotary positions and dropout as a decoder around the MSDA operator calls them.

A case is one pass through one operator: the call alone (inference), or the call and its
gradients (training). ``listed()`` names the cases, ``draw()`` gives more of the same
ranges, ``prepare()`` makes a case's inputs on the GPU, ``run()`` is one pass, ``work()``
the bytes and operations that no implementation can do without, and ``exact()`` the
results in 64 bits. With ``own`` false, ``run`` computes the operators in elementary
torch operations; with ``own`` true it calls this package's operators.
"""

from __future__ import annotations

import math
import random
from typing import Any

import numpy as np
import torch
from torch import Tensor

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _attention(name: str, kind: str, batch: int, queries: int, keys: int, heads: int, channels: int, dtype: str,
               **options: Any) -> dict[str, Any]:
    """``mask``: ``none``; ``boxes``, a bool mask of one box of the image per query, some
    queries with none; ``bias``, an additive mask of distances. ``ragged``: the images'
    states are padded to ``keys``, their lengths spread evenly from a quarter of it."""
    case = {"name": name, "op": "attention", "kind": kind, "batch": batch, "queries": queries, "keys": keys,
            "heads": heads, "kv_heads": heads, "channels": channels, "dtype": dtype, "mask": "none", "ragged": False}
    case.update(options)
    return case


def _rotary(name: str, kind: str, batch: int, grid: str, heads: int, channels: int, sections: str, dtype: str,
            **options: Any) -> dict[str, Any]:
    """``grid``: frames x height x width of the tokens. ``sections``: rotated pairs of
    each axis. ``first``: the first frame's time."""
    case = {"name": name, "op": "rotary", "kind": kind, "batch": batch, "grid": grid, "heads": heads,
            "channels": channels, "sections": sections, "dtype": dtype, "interleaved": False, "first": 0,
            "per_image": False}
    case.update(options)
    return case


def _dropout(name: str, rows: int, width: int, dtype: str, p: float, **options: Any) -> dict[str, Any]:
    case = {"name": name, "op": "dropout", "kind": "train", "rows": rows, "width": width, "dtype": dtype, "p": p,
            "residual": True}
    case.update(options)
    return case


def listed() -> list[dict[str, Any]]:
    return [
        # Object queries of one image over the coarsest level of its pyramid, in a
        # serving loop: a small call, where latency and launches count.
        _attention("queries-infer", "infer", 1, 300, 850, 8, 32, "f16"),
        # One new token of eight captions over their images' encoder states, of padded
        # lengths and shared key heads: bound by reading the states.
        _attention("token-infer", "infer", 8, 1, 21504, 16, 64, "bf16", kv_heads=4, ragged=True),
        # A Mask2Former decoder layer's masked attention over the finest level of
        # 1024 x 1024 images, in training.
        _attention("masked-train", "train", 4, 100, 16384, 8, 32, "bf16", mask="boxes"),
        # Every position of a 1024 x 1024 pixel decoder's pyramid reads a prompt of
        # text states: long queries, few keys.
        _attention("prompt-train", "train", 2, 21504, 77, 8, 64, "bf16"),
        # Two images' finest levels exchange information: both sides long, bound by the
        # matrix cores, at inference and in training.
        _attention("dense-infer", "infer", 2, 16384, 16384, 8, 128, "bf16"),
        _attention("dense-train", "train", 2, 16384, 4096, 8, 64, "f16"),
        # Odd sizes in full precision: an additive distance mask, shared key heads,
        # heads that are no power of two.
        _attention("ragged-train-f32", "train", 3, 301, 1333, 6, 80, "f32", kv_heads=2, mask="bias", ragged=True),
        # The rotary positions of one decoded token of a long video.
        _rotary("rotary-token", "infer", 1, "1x1x1", 16, 64, "8,12,12", "bf16", first=100003),
        # A training step's video clip, 16 frames of 64 x 64 tokens.
        _rotary("rotary-video-train", "train", 2, "16x64x64", 16, 128, "16,24,24", "bf16"),
        # An odd crop in full precision, with a part of the features rotated.
        _rotary("rotary-crop-train", "train", 3, "1x75x97", 8, 32, "0,5,6", "f32", interleaved=True, per_image=True),
        # A decoder layer's queries, four images, before the residual's addition.
        _dropout("dropout-queries", 1200, 256, "f32", 0.1),
        # The hidden features of a pixel decoder's feed-forward part.
        _dropout("dropout-hidden", 86016, 1024, "bf16", 0.1, residual=False),
    ]


def _log(rng: random.Random, low: float, high: float) -> int:
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def _draw_attention(rng: random.Random) -> dict[str, Any]:
    kind = rng.choice(["token", "infer", "train", "train"])
    kv_heads = rng.choice([1, 2, 4, 8])
    mask = rng.choice(["none", "none", "boxes", "bias"])
    queries = rng.randint(1, 8) if kind == "token" else _log(rng, 30, 22000)
    return _attention(
        "", "train" if kind == "train" else "infer", rng.randint(1, 8), queries, _log(rng, 60, 22000),
        kv_heads * rng.choice([1, 1, 2, 3, 4]), rng.choice([16, 32, 32, 64, 64, 80, 96, 128]),
        rng.choice(["bf16", "bf16", "f16", "f32"]), kv_heads=kv_heads, mask=mask, ragged=rng.random() < 0.4)


def _draw_rotary(rng: random.Random) -> dict[str, Any]:
    channels = rng.choice([32, 64, 80, 128])
    share = channels // rng.choice([4, 6, 8, 12])
    grid = (_log(rng, 1, 16), rng.randint(1, 100), rng.randint(1, 100))
    return _rotary(
        "", rng.choice(["infer", "train"]), rng.randint(1, 3), "x".join(map(str, grid)), rng.choice([1, 4, 8, 16]),
        channels, f"{rng.randint(0, share // 2)},{share // 2},{rng.randint(1, share // 2 + 1)}",
        rng.choice(["bf16", "f16", "f32"]), interleaved=rng.random() < 0.4, first=rng.choice([0, 0, _log(rng, 10, 1e6)]),
        per_image=rng.random() < 0.3)


def _draw_dropout(rng: random.Random) -> dict[str, Any]:
    return _dropout("", _log(rng, 1, 90000), rng.randint(3, 1100), rng.choice(["bf16", "f16", "f32"]),
                    rng.choice([0.1, 0.1, 0.25, 0.5, 0.9]), residual=rng.random() < 0.7)


def draw(rng: random.Random) -> dict[str, Any]:
    makers = {"attention": _draw_attention, "rotary": _draw_rotary, "dropout": _draw_dropout}
    op = rng.choice(["attention", "attention", "attention", "rotary", "dropout"])
    while True:
        case = makers[op](rng)
        if op == "attention":
            # At most the pairs of the largest cases of a kind (an eighth in 32 bits, whose
            # products run at another rate), and an additive mask of at most 1 GB.
            each = case["heads"] * case["queries"] * case["keys"]
            pairs = case["batch"] * each * (8 if case["dtype"] == "f32" else 1)
            small = pairs <= (2**30 if case["kind"] == "train" else 2**32)
            small = small and (case["mask"] != "bias" or each <= 2**28)
        else:
            largest = 2 * 2 * 2 * 65536 * 16 * 128 * 2 if op == "rotary" else 5 * 86016 * 1024 * 2
            small = work(case)["bytes"] <= largest
        if small:
            del case["name"]
            return case


# Sizes.


def _lengths(case: dict[str, Any]) -> list[int]:
    """The encoder states of each image."""
    B, S = case["batch"], case["keys"]
    if not case["ragged"]:
        return [S] * B
    return [S - (S - S // 4) * i // max(B - 1, 1) for i in range(B)]


def _grid(case: dict[str, Any]) -> tuple[int, int, int]:
    frames, height, width = (int(n) for n in case["grid"].split("x"))
    return frames, height, width


def _sections(case: dict[str, Any]) -> list[int]:
    return [int(n) for n in case["sections"].split(",")]


def work(case: dict[str, Any]) -> dict[str, float]:
    size = DTYPES[case["dtype"]].itemsize
    train = case["kind"] == "train"
    if case["op"] == "attention":
        B, Q, S, H, D = (case[k] for k in ("batch", "queries", "keys", "heads", "channels"))
        states = sum(_lengths(case))
        q = B * Q * H * D * size
        kv = 2 * states * case["kv_heads"] * D * size
        mask = {"none": 0, "boxes": B * Q * S, "bias": H * Q * S * 4}[case["mask"]]
        # Boxes leave a quarter of the pairs (half of each side, on average).
        pairs = Q * states * H * (0.25 if case["mask"] == "boxes" else 1)
        if not train:
            return {"bytes": 2 * q + kv + mask, "flops": 4.0 * pairs * D}
        return {"bytes": 2 * q + kv + mask + 4 * q + 2 * kv + mask, "flops": 14.0 * pairs * D}
    if case["op"] == "rotary":
        frames, height, width = _grid(case)
        tokens = case["batch"] * frames * height * width
        passes = 2 if train else 1
        elements = tokens * case["heads"] * case["channels"]
        pairs = tokens * case["heads"] * sum(_sections(case))
        positions = (tokens if case["per_image"] else tokens // case["batch"]) * 3 * 8
        return {"bytes": passes * (2 * elements * size + positions), "flops": passes * 6.0 * pairs}
    elements = case["rows"] * case["width"]
    return {"bytes": (5 if case["residual"] else 4) * elements * size, "flops": 4.0 * elements}


# Inputs.


def _boxes(B: int, Q: int, S: int, g: torch.Generator) -> Tensor:
    """``(B, 1, Q, S)``: the positions inside each query's box; every 16th query has none."""
    width = max(1, math.isqrt(S))
    height = -(-S // width)
    position = torch.arange(S, device="cuda")
    y, x = position // width, position % width
    side = 0.25 + 0.5 * torch.rand(2, B, Q, 1, generator=g, device="cuda")
    corner = torch.rand(2, B, Q, 1, generator=g, device="cuda") * (1 - side)
    inside = (y >= corner[0] * height) & (y < (corner[0] + side[0]) * height)
    inside &= (x >= corner[1] * width) & (x < (corner[1] + side[1]) * width)
    inside[:, 15::16] = False
    return inside[:, None]


def _bias(H: int, Q: int, S: int) -> Tensor:
    """``(1, H, Q, S)``: minus the distance of the two places, by a slope for each head."""
    distance = (torch.arange(Q, device="cuda") * (S / Q))[:, None] - torch.arange(S, device="cuda")
    slopes = 2.0 ** (-8.0 * (torch.arange(H, device="cuda") + 1) / H)
    return -(slopes[:, None, None] * distance.abs())[None]


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    train = case["kind"] == "train"

    def normal(*shape: int) -> Tensor:
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    state: dict[str, Any] = {"case": case}
    if case["op"] == "attention":
        B, Q, S, H, D = (case[k] for k in ("batch", "queries", "keys", "heads", "channels"))
        state["q"] = normal(B, Q, H, D).requires_grad_(train)
        state["k"] = normal(B, S, case["kv_heads"], D).requires_grad_(train)
        state["v"] = normal(B, S, case["kv_heads"], D).requires_grad_(train)
        state["mask"] = {"none": lambda: None, "boxes": lambda: _boxes(B, Q, S, g),
                         "bias": lambda: _bias(H, Q, S)}[case["mask"]]()
        state["lengths"] = torch.tensor(_lengths(case), device="cuda") if case["ragged"] else None
        if train:
            state["grad"] = normal(B, Q, H * D)
    elif case["op"] == "rotary":
        B, H, D = case["batch"], case["heads"], case["channels"]
        frames, height, width = _grid(case)
        t, y, x = torch.meshgrid(torch.arange(frames, device="cuda") + case["first"],
                                 torch.arange(height, device="cuda"), torch.arange(width, device="cuda"), indexing="ij")
        positions = torch.stack([t.flatten(), y.flatten(), x.flatten()], -1)
        if case["per_image"]:  # each image a crop at its own place
            shift = torch.randint(0, 1000, (B, 1, 3), generator=g, device="cuda")
            positions = positions + shift
        pairs = sum(_sections(case))
        ladder = torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs
        state.update(x=normal(B, frames * height * width, H, D).requires_grad_(train), positions=positions,
                     frequencies=(10000.0 ** -ladder).float(), sections=tuple(_sections(case)))
        if train:
            state["grad"] = normal(*state["x"].shape)
    else:
        shape = (case["rows"], case["width"])
        state["x"] = normal(*shape).requires_grad_(True)
        state["residual"] = normal(*shape).requires_grad_(True) if case["residual"] else None
        state["grad"] = normal(*shape)
        rng = random.Random(seed)
        state["seed"], state["offset"] = rng.getrandbits(63), rng.getrandbits(40)
    return state


# The operators.


def run(state: dict[str, Any]) -> Any:
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    with torch.no_grad():
        return _PLAIN[op](state)


def _own_attention(state: dict[str, Any]) -> Any:
    from deformops_amd.registry import cross_attention

    q, k, v = state["q"], state["k"], state["v"]
    out = cross_attention(q, k, v, mask=state["mask"], key_lengths=state["lengths"])
    if "grad" not in state:
        return out
    return {"out": out.detach(), **dict(zip("qkv", torch.autograd.grad(out, (q, k, v), state["grad"])))}


def _own_rotary(state: dict[str, Any]) -> Any:
    from deformops_amd.registry import rotary

    out = rotary(state["x"], state["positions"], state["frequencies"], sections=state["sections"],
                 interleaved=state["case"]["interleaved"])
    if "grad" not in state:
        return out
    return {"out": out.detach(), "x": torch.autograd.grad(out, state["x"], state["grad"])[0]}


def _own_dropout(state: dict[str, Any]) -> Any:
    from deformops_amd.registry import dropout

    leaves = {name: state[name] for name in ("x", "residual") if state[name] is not None}
    out = dropout(state["x"], state["case"]["p"], seed=state["seed"], offset=state["offset"],
                  residual=state["residual"])
    return {"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, tuple(leaves.values()), state["grad"])))}


_OWN = {"attention": _own_attention, "rotary": _own_rotary, "dropout": _own_dropout}


# The plain forms: elementary operations in 32 bits.


def _heads_first(x: Tensor, heads: int) -> Tensor:
    """``(B, N, K, D)`` as float32 ``(B, heads, N, D)``, each head repeated for its group."""
    return x.float().repeat_interleave(heads // x.shape[2], 2).transpose(1, 2)


def _plain_attention(state: dict[str, Any]) -> Any:
    case = state["case"]
    B, Q, S, H, D = (case[k] for k in ("batch", "queries", "keys", "heads", "channels"))
    K = case["kv_heads"]
    scale = 1.0 / math.sqrt(D)
    q, k, v = _heads_first(state["q"], H), _heads_first(state["k"], H), _heads_first(state["v"], H)
    scores = torch.matmul(q, k.transpose(2, 3)) * scale
    if case["mask"] == "bias":
        scores = scores + state["mask"]
    elif case["mask"] == "boxes":
        scores = scores.masked_fill(~state["mask"], -math.inf)
    if state["lengths"] is not None:
        beyond = torch.arange(S, device="cuda") >= state["lengths"][:, None, None, None]
        scores = scores.masked_fill(beyond, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(weights, v)
    result = out.transpose(1, 2).reshape(B, Q, H * D).to(state["q"].dtype)
    if "grad" not in state:
        return result
    grad = state["grad"].float().view(B, Q, H, D).transpose(1, 2)
    grad_v = torch.matmul(weights.transpose(2, 3), grad)
    grad_scores = torch.matmul(grad, v.transpose(2, 3)) - (grad * out).sum(-1, keepdim=True)
    grad_scores = weights * grad_scores * scale
    grad_q = torch.matmul(grad_scores, k).transpose(1, 2)
    grad_k = torch.matmul(grad_scores.transpose(2, 3), q)

    def shared(x: Tensor) -> Tensor:  # the sum over the heads of a group
        return x.reshape(B, K, H // K, S, D).sum(2).transpose(1, 2).to(state["k"].dtype).contiguous()

    return {"out": result, "q": grad_q.to(state["q"].dtype).contiguous(), "k": shared(grad_k), "v": shared(grad_v)}


def _rotate(x: Tensor, cos: Tensor, sin: Tensor, interleaved: bool) -> Tensor:
    """The pairs of ``x`` ``(B, L, H, D)`` turned by the angles of ``cos`` and ``sin`` ``(B or 1, L, 1, R)``."""
    pairs = cos.shape[-1]
    first = x[..., 0:2 * pairs:2] if interleaved else x[..., :pairs]
    second = x[..., 1:2 * pairs:2] if interleaved else x[..., pairs:2 * pairs]
    turned = (first * cos - second * sin, second * cos + first * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _angles(state: dict[str, Any]) -> Tensor:
    """``(B or 1, L, 1, R)`` in 64 bits: far positions lose their angle in 32."""
    axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(state["sections"], device="cuda"))
    positions = state["positions"] if state["positions"].dim() == 3 else state["positions"][None]
    return (positions.double()[..., axis] * state["frequencies"].double())[:, :, None]


def _plain_rotary(state: dict[str, Any]) -> Any:
    angles = _angles(state)
    cos, sin = torch.cos(angles).float(), torch.sin(angles).float()
    x, interleaved = state["x"], state["case"]["interleaved"]
    out = _rotate(x.float(), cos, sin, interleaved).to(x.dtype)
    if "grad" not in state:
        return out
    return {"out": out, "x": _rotate(state["grad"].float(), cos, -sin, interleaved).to(x.dtype)}


def _kept(elements: int, p: float, seed: int, offset: int) -> Tensor:
    """Which elements stay: words of Philox4x32 with 7 rounds (Salmon et al., SC 2011),
    the counter (element // 4, offset) and the key ``seed``, against ``p``."""
    word = 0xFFFFFFFF
    block = torch.arange(-(-elements // 4), dtype=torch.int64, device="cuda")
    c = [block & word, block >> 32, torch.full_like(block, offset & word), torch.full_like(block, offset >> 32)]
    key = [seed & word, seed >> 32]
    for _ in range(7):
        low, high = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # modulo 2^64; the shifts below are masked
        c = [((high >> 32) & word) ^ c[1] ^ key[0], high & word, ((low >> 32) & word) ^ c[3] ^ key[1], low & word]
        key = [(key[0] + 0x9E3779B9) & word, (key[1] + 0xBB67AE85) & word]
    threshold = min(round(p * 2**32), word)
    return torch.stack(c, -1).flatten()[:elements] >= threshold


def _plain_dropout(state: dict[str, Any]) -> Any:
    x, p = state["x"], state["case"]["p"]
    keep = _kept(x.numel(), p, state["seed"], state["offset"]).view(x.shape)
    scale = 1.0 / (1.0 - p)
    out = torch.where(keep, x.float() * scale, 0.0)
    if state["residual"] is not None:
        out = out + state["residual"].float()
    result = {"out": out.to(x.dtype), "x": torch.where(keep, state["grad"].float() * scale, 0.0).to(x.dtype)}
    if state["residual"] is not None:
        result["residual"] = state["grad"].clone()
    return result


_PLAIN = {"attention": _plain_attention, "rotary": _plain_rotary, "dropout": _plain_dropout}


# The results in 64 bits.


def _exact_attention(case: dict[str, Any], state: dict[str, Any]) -> Any:
    """One image and head at a time, as softmax and its Jacobian are defined."""
    B, Q, S, H, D = (case[k] for k in ("batch", "queries", "keys", "heads", "channels"))
    group = H // case["kv_heads"]
    train = case["kind"] == "train"
    out = torch.zeros(B, Q, H, D, dtype=torch.float64, device="cuda")
    grads = {name: torch.zeros(state[name].shape, dtype=torch.float64, device="cuda") for name in ("q", "k", "v")}
    for b, length in enumerate(_lengths(case)):
        for h in range(H):
            q, k, v = (state[n][b, :rows, head].double() for n, rows, head in
                       (("q", Q, h), ("k", length, h // group), ("v", length, h // group)))
            logits = q @ k.T / D**0.5
            if case["mask"] == "bias":
                logits += state["mask"][0, h, :, :length].double()
            elif case["mask"] == "boxes":
                logits[~state["mask"][b, 0, :, :length]] = -math.inf
            lse = torch.logsumexp(logits, 1, keepdim=True)
            probability = torch.exp(logits - lse).nan_to_num_(nan=0.0)  # a row without keys
            out[b, :, h] = probability @ v
            if train:
                grad = state["grad"][b].view(Q, H, D)[:, h].double()
                grads["v"][b, :length, h // group] += probability.T @ grad
                slope = grad @ v.T
                slope = probability * (slope - (probability * slope).sum(1, keepdim=True)) / D**0.5
                grads["q"][b, :, h] = slope @ k
                grads["k"][b, :length, h // group] += slope.T @ q
    out = out.view(B, Q, H * D)
    return {"out": out, **grads} if train else out


def _exact_rotary(case: dict[str, Any], state: dict[str, Any]) -> Any:
    """Each pair as a complex number times ``exp(i angle)``."""
    sections = _sections(case)
    pairs = sum(sections)
    position = state["positions"].double()
    angle = torch.cat([position[..., a:a + 1].expand(*position.shape[:-1], n) for a, n in enumerate(sections)], -1)
    angle = (angle * state["frequencies"].double()).unsqueeze(-2)
    turn = torch.complex(angle.cos(), angle.sin())

    def turned(x: Tensor, by: Tensor) -> Tensor:
        x = x.detach().double()
        split = x[..., :2 * pairs]
        split = split.unflatten(-1, (pairs, 2)) if case["interleaved"] else split.unflatten(-1, (2, pairs)).mT
        both = torch.view_as_real(torch.view_as_complex(split.contiguous()) * by)
        both = both.flatten(-2) if case["interleaved"] else both.mT.flatten(-2)
        return torch.cat([both, x[..., 2 * pairs:]], -1)

    out = turned(state["x"], turn)
    return {"out": out, "x": turned(state["grad"], turn.conj())} if case["kind"] == "train" else out


def _exact_kept(elements: int, p: float, seed: int, offset: int) -> Tensor:
    """The generator on unsigned numpy words, its state as (left, right) pairs."""
    mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    kept = np.empty(-(-elements // 4) * 4, dtype=bool)
    chunk = 1 << 20
    for start in range(0, elements, 4 * chunk):
        counter = np.arange(start // 4, min(start // 4 + chunk, kept.size // 4), dtype=np.uint64)
        x0, x1 = counter & mask, counter >> shift
        x2, x3 = (np.full_like(counter, n) for n in (offset % 2**32, offset // 2**32))
        for turn in range(7):
            k0, k1 = ((k + turn * w) % 2**32 for k, w in ((seed % 2**32, 0x9E3779B9), (seed // 2**32, 0xBB67AE85)))
            a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
            x0, x1, x2, x3 = (b >> shift) ^ x1 ^ np.uint64(k0), b & mask, (a >> shift) ^ x3 ^ np.uint64(k1), a & mask
        words = np.stack([x0, x1, x2, x3], 1).reshape(-1)
        kept[start:start + words.size] = words / 2**32 >= min(round(p * 2**32), 2**32 - 1) / 2**32
    return torch.from_numpy(kept[:elements]).cuda()


def _exact_dropout(case: dict[str, Any], state: dict[str, Any]) -> Any:
    keep = _exact_kept(state["x"].numel(), case["p"], state["seed"], state["offset"]).view(state["x"].shape).double()
    scale = keep / (1 - case["p"])
    out = state["x"].detach().double() * scale
    result = {"out": out, "x": state["grad"].double() * scale}
    if case["residual"]:
        result["out"] = out + state["residual"].detach().double()
        result["residual"] = state["grad"].double()
    return result


def exact(case: dict[str, Any], seed: int) -> Any:
    state = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "rotary": _exact_rotary, "dropout": _exact_dropout}[case["op"]](case, state)
