"""The f32 results of the dense projection, whose bound in the other tests holds
for any inputs and grows with the columns.

A step of 16 columns may truncate its chain's sum, a unit of 2^-23 at most.
After j of n steps that sum has sqrt(j / n) of its norm in the end, and the mean
of those is 2/3: n * 2/3 * 2^-23 of a chain's norm.  The 4096 columns are 256
steps in one chain (2.04e-5; 4.4e-6 is what they lose), 128 in each of two
(128 x 128 tiles), 64 in each of four (up to 64 tokens: 5.1e-6 and 1.0e-6), whose
losses do not add up faster than their squares.  A cluster's shares are
shorter.  Sums rounded to bf16 on their way would leave about 1e-3."""

from __future__ import annotations

import pytest
import torch

U = 2.0**-24


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,tokens", [
    (2688, 1), (1200, 19), (20000, 33), (96, 64),           # up to 64 tokens, a tile's columns shared or not
    (2688, 100), (8000, 300), (3700, 380), (10000, 300),    # 128 x 128, 128 x 256, shared or not
    (2600, 401), (3712, 512), (3700, 1000), (5000, 3001)])  # pairs, shared or not
def test_projection_sums(k, cuda, rows, tokens):
    steps = 256 if tokens > 64 else 64  # of the longest chain that the tile may have
    g = torch.Generator(device=cuda).manual_seed(rows)
    W, x = (torch.randn(n, 4096, generator=g, device=cuda).bfloat16() for n in (rows, tokens))
    out = torch.empty(tokens, rows, device=cuda)
    k.linear_bf16(out, W, x, rows, 4096, tokens)
    want = x.double() @ W.double().t()
    off = float((out.double() - want).norm() / want.norm())
    assert off <= steps * 2 / 3 * 2.0**-23 + 4 * U, off
