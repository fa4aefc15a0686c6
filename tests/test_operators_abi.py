"""Host-side refusals and workspace sizes of the C entries for cross attention, rotary positions
and dropout. Nothing is launched: every call here ends at a check, or asks for sizes."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

from deformops_amd.backends.hip import _lib

F32, F16, BF16 = 0, 1, 2
OK, INVALID, UNSUPPORTED = 0, 1, 2
P, L = ctypes.c_void_p, ctypes.c_int64
SOME = 1 << 20  # an address that no call may read


class Attention(ctypes.Structure):
    _fields_ = [(n, P) for n in ("query", "key", "value", "mask", "key_lengths", "output")] + [
        ("query_strides", L * 3), ("key_strides", L * 3), ("value_strides", L * 3), ("mask_strides", L * 4),
        *((n, L) for n in ("batch", "queries", "keys", "heads", "key_heads", "channels")), ("scale", ctypes.c_float),
        *((n, ctypes.c_int) for n in ("dtype", "mask_kind", "mask_dtype", "index_dtype"))]


@pytest.fixture(scope="module")
def lib():
    out = _lib.load().cdll
    out.deformops_last_error.restype = ctypes.c_char_p
    return out


def attention(B=2, Q=300, S=500, H=8, K=8, D=32, dtype=BF16, **changes) -> Attention:  # noqa: N803
    """Dense operands."""
    call = Attention(query=SOME, key=SOME, value=SOME, output=SOME, batch=B, queries=Q, keys=S, heads=H, key_heads=K,
                     channels=D, scale=0.5, dtype=dtype, query_strides=(L * 3)(Q * H * D, H * D, D),
                     key_strides=(L * 3)(S * K * D, K * D, D), value_strides=(L * 3)(S * K * D, K * D, D))
    for name, value in changes.items():
        setattr(call, name, value)
    return call


def sizes_of(lib, call):
    forward, backward = L(-1), L(-1)
    status = lib.deformops_cross_attention_workspace_size(ctypes.byref(call), ctypes.byref(forward), ctypes.byref(backward))
    return status, forward.value, backward.value


def forward(lib, call, workspace=None, size=0):
    return lib.deformops_cross_attention_forward(ctypes.byref(call), None, P(workspace), L(size), None)


def backward(lib, call, workspace=None, size=0, grad=SOME, grads=(SOME, SOME, SOME), stats=SOME):
    return lib.deformops_cross_attention_backward(ctypes.byref(call), P(stats), P(grad), *(P(g) for g in grads),
                                                  P(workspace), L(size), None)


def test_every_declared_function_is_exported_and_bound(lib):
    header = Path(__file__).resolve().parents[1] / "include" / "deformops_amd.h"
    declared = re.findall(r"^(?:int|const char\*)\s+(deformops_\w+)\(", header.read_text(), flags=re.M)
    assert set(declared) == set(_lib.OPERATOR_SYMBOLS)
    for name in declared:
        assert getattr(lib, name).argtypes is not None


def test_the_structure_is_the_headers(lib):
    """A call that the header's layout reads otherwise would be refused here, or given other sizes."""
    assert ctypes.sizeof(Attention) == 6 * 8 + 13 * 8 + 6 * 8 + 4 * 5 + 4
    assert sizes_of(lib, attention(B=64)) == (OK, 0, 64 * 8 * 300 * 4)  # delta alone


REFUSED = {
    "dtype": ({"dtype": 7}, INVALID, b"dtype"),
    "negative": ({"queries": -1}, INVALID, b"negative"),
    "no channels": ({"channels": 0}, INVALID, b"channels"),
    "groups of heads": ({"key_heads": 3}, INVALID, b"multiple"),
    "wide heads": ({"channels": 129}, UNSUPPORTED, b"128"),
    "scale": ({"scale": 0.0}, INVALID, b"scale"),
    "infinite scale": ({"scale": float("inf")}, INVALID, b"scale"),
    "scale nan": ({"scale": float("nan")}, INVALID, b"scale"),
    "mask kind": ({"mask_kind": 3}, INVALID, b"mask"),
    "mask dtype": ({"mask_kind": 2, "mask_dtype": 9}, INVALID, b"mask"),
    "lengths": ({"key_lengths": SOME, "index_dtype": 9}, INVALID, b"key_lengths"),
    "many queries": ({"queries": 1 << 31}, UNSUPPORTED, b"2^31"),
    "many rows of a group": ({"queries": 1 << 29, "key_heads": 1}, UNSUPPORTED, b"2^31"),
}


@pytest.mark.parametrize("name", REFUSED)
def test_attention_refusals(lib, name):
    changes, status, words = REFUSED[name]
    call = attention(**changes)
    for got in (sizes_of(lib, call)[0], forward(lib, call), backward(lib, call)):
        assert got == status and words in lib.deformops_last_error()


def test_attention_pointers_and_workspaces(lib):
    assert forward(lib, attention(query=None)) == INVALID and b"null" in lib.deformops_last_error()
    assert forward(lib, attention(value=None)) == INVALID
    assert forward(lib, attention(mask_kind=1)) == INVALID  # no mask
    assert lib.deformops_cross_attention_workspace_size(None, None, None) == INVALID
    assert lib.deformops_cross_attention_workspace_size(ctypes.byref(attention()), None, None) == INVALID
    few = attention(B=1, Q=1, S=9000)  # in pieces
    status, first, second = sizes_of(lib, few)
    assert status == OK and first > 0 and second > 0
    for got in (forward(lib, few), forward(lib, few, SOME, first - 1), forward(lib, few, SOME + 8, first),
                backward(lib, few), backward(lib, few, SOME, second - 1), backward(lib, few, SOME + 8, second)):
        assert got == INVALID and b"workspace" in lib.deformops_last_error()
    assert backward(lib, few, SOME, second, stats=None) == INVALID
    assert backward(lib, few, SOME, second, grads=(SOME, None, SOME)) == INVALID
    assert backward(lib, few, SOME, second, grad=SOME + 2) == INVALID and b"aligned" in lib.deformops_last_error()
    # Nothing to do: no tensor, and no workspace, is asked for.
    assert forward(lib, attention(B=0, query=None)) == OK
    assert forward(lib, attention(Q=0, output=None, mask_kind=1)) == OK
    assert backward(lib, attention(Q=0, S=0)) == OK


def test_attention_calls_that_pass_a_grid(lib):
    """2^24 workgroups of 256 threads are one too many; refused before anything is launched."""
    whole = 1 << 60
    for call in (attention(B=1024, Q=1 << 22, H=1, K=1), attention(B=1024, Q=1 << 24, H=1, K=1, mask_kind=0)):
        assert forward(lib, call, SOME, whole) == UNSUPPORTED and b"grid" in lib.deformops_last_error()
        assert backward(lib, call, SOME, whole) == UNSUPPORTED and b"grid" in lib.deformops_last_error()
    keys = attention(B=1024, Q=1, S=1 << 22, H=1, K=1)
    assert backward(lib, keys, SOME, whole) == UNSUPPORTED
    # Operands that have to be packed: rows off 16 bytes, a mask in another order.
    odd = attention(B=1, Q=1 << 30, S=4, H=8, K=8, query=SOME + 2)
    assert forward(lib, odd, SOME, whole) == UNSUPPORTED
    mask = attention(B=1, Q=1 << 20, S=1 << 13, H=1, K=1, mask=SOME, mask_kind=2, mask_dtype=F32,
                     mask_strides=(L * 4)(0, 0, 1, 1 << 20))
    assert forward(lib, mask, SOME, whole) == UNSUPPORTED and b"grid" in lib.deformops_last_error()


def rotary(lib, *, dtype=F32, position_type=0, x=SOME, y=SOME, sections=(4, 4), batch=2, tokens=10, heads=4, channels=16,
           positions=SOME, frequencies=SOME, strides=(640, 64, 16)):
    return lib.deformops_rotary(P(x), (L * 3)(*strides), P(y), dtype, P(positions), (L * 3)(0, 2, 1), position_type,
                                P(frequencies), (L * max(1, len(sections)))(*sections), L(len(sections)), L(batch),
                                L(tokens), L(heads), L(channels), 0, 0, None)


@pytest.mark.parametrize(("changes", "status", "words"), [
    ({"dtype": 5}, INVALID, b"dtype"),
    ({"position_type": 4}, INVALID, b"positions"),
    ({"position_type": -1}, INVALID, b"positions"),
    ({"sections": ()}, INVALID, b"axes"),
    ({"sections": (4, -1)}, INVALID, b"section"),
    ({"sections": (8, 1)}, INVALID, b"rotate"),
    ({"sections": (200, 57), "channels": 1024}, UNSUPPORTED, b"256"),
    ({"tokens": -1}, INVALID, b"negative"),
    ({"heads": 1 << 11, "channels": 1 << 10}, UNSUPPORTED, b"2^20"),
    ({"x": None}, INVALID, b"null"),
    ({"positions": None}, INVALID, b"null"),
    ({"batch": 1 << 24, "tokens": 1 << 20}, UNSUPPORTED, b"grid"),
    ({"batch": 1 << 40, "tokens": 1 << 22}, UNSUPPORTED, b"grid"),
], ids=lambda c: "-".join(c) if isinstance(c, dict) else None)
def test_rotary_refusals(lib, changes, status, words):
    assert rotary(lib, **changes) == status and words in lib.deformops_last_error()


def test_rotary_calls_without_elements(lib):
    for name in ("batch", "tokens", "heads"):
        assert rotary(lib, x=None, y=None, **{name: 0}) == OK


@pytest.mark.parametrize(("dtype", "elements", "p", "x", "status"), [
    (4, 10, 0.5, SOME, INVALID), (F32, -1, 0.5, SOME, INVALID), (F32, 10, 1.5, SOME, INVALID),
    (F32, 10, -0.1, SOME, INVALID), (F32, 10, float("nan"), SOME, INVALID), (F32, 10, 0.5, None, INVALID),
    (F32, 0, 0.5, None, OK),
])
def test_dropout_refusals(lib, dtype, elements, p, x, status):
    assert lib.deformops_dropout(P(x), None, P(SOME), dtype, L(elements), ctypes.c_double(p), ctypes.c_uint64(1), None,
                                 ctypes.c_uint64(0), None) == status
