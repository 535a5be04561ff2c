"""The precision that the chunked scan states, on inputs where a lost part would show.

The bounds of the other tests hold for any inputs and grow with the length of a
sum; here the inputs leave the sums one term, or let their terms cancel, and
the bounds are the parts' own:

  * The states' new terms d x B: x d is split into three bf16 numbers, each of
    which leaves at most 2^-8 of what it is given: together they hold all 24 bits.
    expf and log1pf of the step, 2 units of 2^-23 each at most, the product x d and
    three sums that may truncate (a unit each) come to less than 20 * 2^-24.
    Two parts would leave up to 2^-16, 256 * 2^-24.
  * The state before a chunk meets C as two bf16 numbers: 2^-16 of each term,
    and sums in f32 that may truncate a unit of 2^-23 for 16 of the 2 d_state
    products, 2^-19 of the sum of magnitudes.  One part would leave up to 2^-8.

They are checked on the CPU too, with the parts left out of a model of the
splits."""

from __future__ import annotations

import pytest
import torch

import hybrid_ref as ref

F32, BF16, U = torch.float32, torch.bfloat16, ref.U


def parts(v, n):
    """The sum of the first n bf16 parts of f32 numbers, exact."""
    out = torch.zeros_like(v, dtype=torch.float64)
    for _ in range(n):
        p = v.bfloat16()
        out += p.double()
        v = v - p.float()
    return out


def test_a_missing_part_of_the_new_terms_would_show():
    g = torch.Generator().manual_seed(0)
    v = torch.randn(10000, generator=g).bfloat16().float() * torch.rand(10000, generator=g)
    off = [float(((parts(v, n) - v.double()) / v.double()).abs().max()) for n in (1, 2, 3)]
    assert off[2] <= 2.0**-27 and off[1] > 30 * U and off[0] > 2.0**-10


def cancelling(heads, n, g):
    """States whose columns cancel in pairs but for a little, and the columns' order."""
    half = torch.randn(heads, 64, n // 2, generator=g)
    return torch.cat([half, -half + 2.0**-9 * torch.randn(half.shape, generator=g)], -1)


def test_a_missing_part_of_the_state_would_show():
    s = cancelling(4, 64, torch.Generator().manual_seed(1))
    want, size = s.double().sum(-1), s.double().abs().sum(-1)
    bound = 2.0**-14 * size + ref.HALF[BF16] * want.abs()
    assert ((parts(s, 2).sum(-1) - want).abs() <= bound).all()
    assert ((parts(s, 1).sum(-1) - want).abs() > bound).float().mean() > 0.2


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,groups", [([128], 2, 1), ([64], 6, 2), ([33, 128, 1, 200], 5, 1), ([1000], 4, 4)])
@pytest.mark.parametrize("d_state", [64, 128])
def test_states_of_a_single_term(k, cuda, lens, heads, groups, d_state):
    g = torch.Generator().manual_seed(sum(lens))
    t, s, p = sum(lens), len(lens), 64
    cu = torch.tensor([0, *lens]).cumsum(0)
    x, b, c = (torch.randn(t, w, generator=g).bfloat16() for w in (heads * p, groups * d_state, groups * d_state))
    dt = torch.randn(t, heads, generator=g).bfloat16()
    keep = torch.tensor([int(cu[i]) + (lens[i] * 5 // 8) for i in range(s)])  # the one token of each with an x
    only = torch.zeros(t, 1, dtype=BF16)
    only[keep] = 1
    x = x * only
    y, state = torch.zeros(t, heads * p, dtype=BF16, device=cuda), torch.zeros(s, heads, p, d_state, device=cuda)
    zero = torch.zeros(heads, device=cuda)
    k.ssm_prompt(y, x.to(cuda), dt.to(cuda), zero, b.to(cuda), c.to(cuda), None, None, state, cu.int().to(cuda), s, t,
                 heads, p, groups, d_state)
    d = ref.softplus(dt[keep].double())
    bs = b[keep].double().view(s, groups, d_state).repeat_interleave(heads // groups, 1)
    new = (d[..., None] * x[keep].double().view(s, heads, p))[..., None] * bs[:, :, None]
    ref.within(state, new, 20 * U * new.abs() + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("d_state", [64, 128])
@pytest.mark.parametrize("tokens", [40, 128, 300])
def test_outputs_of_a_carried_state_that_cancels(k, cuda, tokens, d_state):
    g = torch.Generator().manual_seed(d_state + tokens)
    heads, p = 4, 64
    s = cancelling(heads, d_state, g)
    c = torch.ones(tokens, d_state).bfloat16()
    y = torch.zeros(tokens, heads * p, dtype=BF16, device=cuda)
    x, dt = torch.zeros(tokens, heads * p, dtype=BF16), torch.zeros(tokens, heads, dtype=BF16)
    state, zero = s[None].to(cuda), torch.zeros(heads, device=cuda)
    k.ssm_prompt(y, x.to(cuda), dt.to(cuda), zero, torch.randn(tokens, d_state, generator=g).bfloat16().to(cuda),
                 c.to(cuda), None, None, state, None, 1, tokens, heads, p, 1, d_state,
                 has_state=torch.tensor([True], device=cuda))
    want, size = s.double().sum(-1).flatten(), s.double().abs().sum(-1).flatten()
    bound = 2.0**-14 * size + ref.HALF[BF16] * want.abs()
    ref.within(y, want.expand(tokens, -1), bound.expand(tokens, -1))
    assert torch.equal(state[0].cpu(), s)  # nothing decays and nothing is added
