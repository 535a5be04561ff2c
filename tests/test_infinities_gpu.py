"""Infinities and NaN in the scan's inputs: they reach what the recurrence lets
them reach, and nothing else."""

from __future__ import annotations

import pytest
import torch

import hybrid_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.parametrize("d_state", [1, 5, 16, 40, 64, 100, 130])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_infinity_with_any_number_of_states(k, cuda, d_state, dtype):
    """All terms positive: the output of an infinite input, and of the tokens behind it, is infinite
    and no NaN, however many columns the kernel pads the state with."""
    g = torch.Generator().manual_seed(d_state)
    t, p = 20, 3
    x, b, c = (torch.rand(t, w, generator=g).to(dtype) + 0.5 for w in (p, d_state, d_state))
    x[7, 1] = INF
    y, state = torch.zeros(t, p, dtype=dtype, device=cuda), torch.zeros(1, 1, p, d_state, device=cuda)
    one = torch.ones(1, device=cuda)
    k.ssm_prompt(y, x.to(cuda), torch.zeros(t, 1, dtype=dtype, device=cuda), -one, b.to(cuda), c.to(cuda), one, None,
                 state, None, 1, t, 1, p, 1, d_state)
    want = torch.zeros(t, p, dtype=torch.bool)
    want[7:, 1] = True
    y = y.float().cpu()
    assert torch.equal(y == INF, want) and not torch.isnan(y).any()
    assert (state[0, 0, 1] == INF).all() and torch.isfinite(state[0, 0, [0, 2]]).all()


@pytest.mark.parametrize("d_state", [4, 28, 32, 48, 64, 100, 132, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_token_infinity_with_any_number_of_states(k, cuda, d_state, dtype):
    p = 3
    ch = p + 2 * d_state
    row = torch.ones(1, ch, dtype=dtype, device=cuda)
    row[0, 1] = INF
    cw = torch.zeros(ch, 2, device=cuda)
    cw[:, 1] = 1
    one = torch.ones(1, device=cuda)
    out = torch.zeros(1, p, dtype=dtype, device=cuda)
    conv, state = torch.zeros(1, 1, ch, dtype=dtype, device=cuda), torch.ones(1, 1, p, d_state, device=cuda)
    k.ssm_token(out, row, torch.zeros(1, 1, dtype=dtype, device=cuda), cw, None, conv, -one, one, None, state, 1, 1, p, 1,
                d_state, 2)
    assert (out[0].float().cpu() == INF).tolist() == [False, True, False] and not torch.isnan(out).any()
    assert (state[0, 0, 1] == INF).all() and torch.isfinite(state[0, 0, [0, 2]]).all()
