"""Packs of many sequences: the work of finding a sequence's tiles grows with
their number, not with its square."""

from __future__ import annotations

import time

import pytest
import torch

import hybrid_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.parametrize("seqs", [31, 32, 33, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_conv(k, cuda, seqs, dtype):
    """Lengths from none to some tiles, at the sizes where the search takes a round more."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 4, (seqs,), generator=g)
    lens[torch.randint(0, seqs, (5,), generator=g)] = 70
    lens[::7] = 0
    cu = torch.zeros(seqs + 1, dtype=torch.int32)
    cu[1:] = lens.cumsum(0)
    t, channels, width = int(cu[-1]) + 3, 8, 4
    x = torch.randn(t, channels, generator=g).to(dtype)
    w, b = torch.randn(channels, width, generator=g), torch.randn(channels, generator=g)
    state = torch.randn(seqs + 2, width - 1, channels, generator=g).to(dtype)
    slots = torch.randperm(seqs + 2, generator=g)[:seqs]
    has = torch.rand(seqs, generator=g) < 0.5
    out, st = torch.full((t, channels), 9.0, dtype=dtype, device=cuda), state.to(cuda)
    k.conv1d_prompt(out, x.to(cuda), w.to(cuda), b.to(cuda), st, cu.to(cuda), seqs, t, channels, width,
                    slots=slots.int().to(cuda), has_state=has.to(cuda))
    want, size, new = ref.conv(x, w, b, state, cu.tolist(), slots.tolist(), has.tolist())
    end = int(cu[-1])
    ref.within(out[:end], want[:end], (ref.HALF[dtype] * want.abs() + 16 * ref.U * size)[:end] + 1e-30)
    assert (out[end:] == 9).all() and torch.equal(st.cpu().double(), new)


def test_conv_of_four_million_sequences(k, cuda):
    """One token of each: a search that walked the offsets took minutes here."""
    seqs, channels = 1 << 22, 1
    x = torch.randn(seqs, channels, device=cuda)
    w, cu = torch.randn(channels, 2, device=cuda), torch.arange(seqs + 1, dtype=torch.int32, device=cuda)
    out = torch.empty_like(x)
    state = torch.zeros(seqs, 1, channels, device=cuda)
    torch.cuda.synchronize()
    began = time.monotonic()
    k.conv1d_prompt(out, x, w, None, state, cu, seqs, seqs, channels, 2, silu=False)
    torch.cuda.synchronize()
    assert time.monotonic() - began < 2
    assert torch.equal(out, x * w[:, 1]) and torch.equal(state[:, 0], x)
