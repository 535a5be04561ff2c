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


def one_token_scan(k, cuda, seqs, lens=None, d_state=64):
    """A pack of `seqs` sequences (one token each, or lens) from zero states, two heads, one group;
    returns what the first token of each gives in 64 bits too."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.ones(seqs, dtype=torch.int64) if lens is None else lens
    cu = torch.zeros(seqs + 1, dtype=torch.int64)
    cu[1:] = lens.cumsum(0)
    t, h, p, n = int(cu[-1]), 2, 64, d_state
    x, b, c = (torch.randn(t, w, generator=g).bfloat16() for w in (h * p, n, n))
    dt, A, D = torch.randn(t, h, generator=g).bfloat16(), -torch.rand(h, generator=g), torch.randn(h, generator=g)
    y, state = torch.full((t, h * p), 9.0, dtype=BF16, device=cuda), torch.full((seqs, h, p, n), 9.0, device=cuda)
    xd, bd, cd, dtd = (v.to(cuda) for v in (x, b, c, dt))
    k.ssm_prompt(y, xd, dtd, A.to(cuda), bd, cd, D.to(cuda), None, state, cu.int().to(cuda), seqs, t, h, p, 1, n)
    first = cu[:-1][lens > 0].to(cuda)
    xs, d = xd[first].double().view(-1, h, p), ref.softplus(dtd[first].double())
    new = (d[..., None] * xs)[..., None] * bd[first].double()[:, None, None]
    parts = new * cd[first].double()[:, None, None]
    want = parts.sum(-1) + D.to(cuda).double()[:, None] * xs
    size = parts.abs().sum(-1) + (D.to(cuda).double()[:, None] * xs).abs()
    return y, state, first, want.flatten(1), size.flatten(1), new


@pytest.mark.parametrize("seqs", [16384, 16385, 40000])
def test_scan(k, cuda, seqs):
    """The most sequences of the chunked form, and more: bf16 as in test_ssm_gpu, P and the output
    rounded by half a step each, chains of 64 columns."""
    y, state, first, want, size, new = one_token_scan(k, cuda, seqs)
    h = ref.HALF[BF16]
    ref.within(y, want.cpu(), (h * (want.abs() + h * size) + (h + 256 * ref.U) * size + 1e-30).cpu())
    ref.within(state, new.cpu(), (32 * ref.U * new.abs() + 1e-30).cpu())


def test_scan_of_sequences_that_are_mostly_empty(k, cuda):
    """Every role steps through 16,000 empty sequences in a row: in time for the others' waits."""
    from ervf_b200 import _lib

    lens = torch.zeros(16384, dtype=torch.int64)
    lens[0], lens[2], lens[16000], lens[16383] = 200, 1, 300, 2
    y, state, first, want, size, new = one_token_scan(k, cuda, 16384, lens)
    h = ref.HALF[BF16]
    ref.within(y[first], want.cpu(), (h * (want.abs() + h * size) + (h + 256 * ref.U) * size + 1e-30).cpu())
    assert (state[(lens == 0).nonzero().flatten().to(cuda)] == 0).all()
    assert _lib.load().ervf_device_status() == _lib.OK
