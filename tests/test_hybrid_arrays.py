"""What the dense and state-space methods take from objects with
``__cuda_array_interface__``: checked as tensors are, before any CUDA call."""

from __future__ import annotations

import pytest
import torch

from ervf_b200 import GPUKernels

AT = 1 << 20


class Array:
    def __init__(self, shape, typestr, strides=None, at=AT):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (at, False), "version": 3,
                                         "strides": strides}


class Launches:
    """Takes the place of the launch: nothing here has a GPU."""

    def __init__(self, monkeypatch):
        self.seen = []
        monkeypatch.setattr(GPUKernels, "_launch", lambda k, name, *args: self.seen.append((name, args)))


@pytest.fixture()
def k():
    return GPUKernels(device="cuda:0")


def calls(k, **over):
    """One call of each method with arrays of the right kind, but for those in `over`."""
    f, u, i, b = (lambda *s: Array(s, "<f4")), (lambda *s: Array(s, "<u2")), (lambda *s: Array(s, "<i4")), \
        (lambda *s: Array(s, "|b1"))
    v = dict(W=u(16, 8), bias=f(16), cw=f(8, 4), cb=f(8), cs=u(2, 3, 8), cu=i(2), slots=i(1), has=b(1), A=f(2), D=f(2),
             dtb=f(2), st=f(2, 2, 2, 4), nw=f(4), tw=f(12, 2), tb=f(12), tcs=u(2, 1, 12))
    v.update(over)
    bf = torch.bfloat16
    return {
        "linear": lambda: k.linear_bf16(AT, v["W"], AT, 16, 8, 3, bias=v["bias"], dtype=bf),
        "conv": lambda: k.conv1d_prompt(AT, AT, v["cw"], v["cb"], v["cs"], v["cu"], 1, 3, 8, 4, slots=v["slots"],
                                        has_state=v["has"], n_slots=2, dtype=bf),
        "scan": lambda: k.ssm_prompt(AT, AT, AT, v["A"], AT, AT, v["D"], v["dtb"], v["st"], v["cu"], 1, 3, 2, 2, 1, 4,
                                     slots=v["slots"], has_state=v["has"], n_slots=2, dtype=bf),
        "token": lambda: k.ssm_token(AT, AT, AT, v["tw"], v["tb"], v["tcs"], v["A"], v["D"], v["dtb"], v["st"], 1, 2, 2,
                                     1, 4, 2, norm_w=v["nw"], slots=v["slots"], n_slots=2, dtype=bf),
        "norm": lambda: k.gated_norm(AT, AT, None, v["nw"], 3, 2, 2, dtype=bf),
    }


def test_arrays_of_the_right_kind_are_taken(k, monkeypatch):
    seen = Launches(monkeypatch).seen
    for call in calls(k).values():
        call()
    assert len(seen) == 5
    calls(k, W=Array((16, 8), "<u2", strides=(16, 2)), bias=Array((1, 16, 1), "<f4", strides=(0, 4, 12)))["linear"]()
    k.gated_norm(Array((3, 4), "<f4", strides=(16, 4)), AT, None, AT, 3, 2, 2)
    assert len(seen) == 7


@pytest.mark.parametrize("name,what,array", [
    ("linear", "W", Array((16, 8), "<f4")), ("linear", "W", Array((16, 8), "<u2", (2, 32))),
    ("linear", "W", Array((16, 8), "<u2", (32, 2))), ("linear", "bias", Array((16,), "<f8")),
    ("linear", "bias", Array((16,), "<f4", (8,))), ("conv", "cw", Array((8, 4), "<u2")),
    ("conv", "cs", Array((2, 3, 8), "<f4")), ("conv", "cu", Array((2,), "<i8")), ("conv", "slots", Array((1,), "<u4")),
    ("conv", "has", Array((1,), "<i4")), ("scan", "A", Array((2,), "<f8")), ("scan", "st", Array((2, 2, 2, 4), "<u2")),
    ("scan", "cu", Array((2,), "<i4", (8,))), ("token", "tcs", Array((2, 1, 12), "<f4")),
    ("token", "D", Array((2,), "<f2")), ("norm", "nw", Array((4,), "<f4", (-4,)))])
def test_arrays_of_another_type_or_order_are_refused(k, monkeypatch, name, what, array):
    """Their bytes would be read as the elements of the right kind."""
    seen = Launches(monkeypatch).seen
    with pytest.raises(ValueError):
        calls(k, **{what: array})[name]()
    assert not seen


def test_rows_are_taken_contiguous(k, monkeypatch):
    Launches(monkeypatch)
    with pytest.raises(ValueError):
        k.gated_norm(Array((3, 4), "<f4", strides=(32, 4)), AT, None, AT, 3, 2, 2)


@pytest.mark.parametrize("stream,handle", [
    (type("Torch", (), {"cuda_stream": 64})(), 64), (type("Cupy", (), {"ptr": 128})(), 128), (256, 256), (0, 0)])
def test_a_stream_of_any_kind(k, monkeypatch, stream, handle):
    from ervf_b200 import _lib

    seen = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(args[-1]))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    k.stream = stream
    k.gated_norm(AT, AT, None, AT, 3, 2, 2, dtype=torch.float32)
    k.mv_bf16(AT, AT, AT, 8, 8)
    assert seen == [handle, handle]


def test_sizes_of_nothing_are_refused_beside_a_state(k):
    state, f32 = torch.zeros(4, 4), torch.float32
    for call in (lambda: k.ssm_prompt(AT, AT, AT, AT, AT, AT, None, None, state, AT, 1, 3, 0, 64, 1, 64, dtype=f32),
                 lambda: k.ssm_token(AT, AT, AT, AT, None, AT, AT, None, None, state, 1, 4, 64, 1, 0, 4, dtype=f32),
                 lambda: k.conv1d_prompt(AT, AT, AT, None, state, AT, 1, 3, 0, 4, dtype=f32)):
        with pytest.raises(ValueError):
            call()


WIDE = 2 ** 32 + 8  # 8 in 32 bits


@pytest.mark.parametrize("size", [WIDE, 2 ** 31, -WIDE])
def test_sizes_that_pass_32_bits_are_refused(k, monkeypatch, size):
    """Cut to 32 bits they would be other sizes, and most of the output would stay as it was."""
    seen = Launches(monkeypatch).seen
    f32 = torch.float32

    def linear(rows=8, cols=8, tokens=3):
        k.linear_bf16(AT, AT, AT, rows, cols, tokens, dtype=f32)

    def conv(seqs=1, tokens=3, channels=8, width=4, n_slots=1):
        k.conv1d_prompt(AT, AT, AT, None, AT, AT, seqs, tokens, channels, width, n_slots=n_slots, dtype=f32)

    def scan(seqs=1, tokens=3, heads=2, head_dim=2, groups=1, d_state=4, n_slots=1):
        k.ssm_prompt(AT, AT, AT, AT, AT, AT, None, None, AT, AT, seqs, tokens, heads, head_dim, groups, d_state,
                     n_slots=n_slots, dtype=f32)

    def token(seqs=1, heads=2, head_dim=2, groups=1, d_state=4, width=4, n_slots=1):
        k.ssm_token(AT, AT, AT, AT, None, AT, AT, None, None, AT, seqs, heads, head_dim, groups, d_state, width,
                    n_slots=n_slots, dtype=f32)

    def norm(tokens=3, groups=1, group_size=8):
        k.gated_norm(AT, AT, None, AT, tokens, groups, group_size, dtype=f32)

    for call in (linear, conv, scan, token, norm):
        for name in call.__code__.co_varnames[:call.__code__.co_argcount]:
            with pytest.raises(ValueError):
                call(**{name: size})
    assert not seen
    for call in (linear, conv, scan, token, norm):
        call()
    assert len(seen) == 5
