"""Every kind of stream that ``GPUKernels.stream`` takes, through the method that also takes scratch
on it."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


class CupyLike:
    def __init__(self, handle):
        self.ptr = handle


@pytest.mark.parametrize("kind", ["torch", "cupy", "handle", "legacy default", "external"])
def test_scan_on_a_stream_of_any_kind(cuda, kind):
    from ervf_b200 import GPUKernels

    side = torch.cuda.Stream()
    g = torch.Generator(device=cuda).manual_seed(1)
    h, n, t = 4, 64, 300
    xbc = torch.randn(t, h * 64 + 2 * n, generator=g, device=cuda).bfloat16()
    dt, one = torch.randn(t, h, generator=g, device=cuda).bfloat16(), torch.ones(h, device=cuda)

    def call(k, y, st):
        k.ssm_prompt(y, xbc[:, :h * 64], dt, -one, xbc[:, h * 64:h * 64 + n], xbc[:, h * 64 + n:], one, None, st, None,
                     1, t, h, 64, 1, n)

    outs = [(torch.zeros(t, h * 64, dtype=torch.bfloat16, device=cuda), torch.zeros(1, h, 64, n, device=cuda))
            for _ in range(2)]
    k = GPUKernels()
    call(k, *outs[0])
    torch.cuda.synchronize()
    handle = side.cuda_stream
    k.stream = {"torch": side, "cupy": CupyLike(handle), "handle": handle, "legacy default": CupyLike(0),
                "external": torch.cuda.ExternalStream(handle)}[kind]
    if kind != "legacy default":
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)  # the call stands behind this on its stream
    call(k, *outs[1])
    if kind != "legacy default":
        torch.cuda.current_stream().synchronize()
        assert not side.query()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
